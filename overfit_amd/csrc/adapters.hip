// adapters.hip — low-rank adapters of many requests beside a shared projection: for every activation row m with an adapter
// slot s, y[m] += scale_s * B_s (A_s x[m]), A_s [rank][in], B_s [out][rank].
//
// Two launches: the rows' products A_s x[m] into scratch planes (shrink), then B_s times them into the outputs (expand). Both
// are matrix products over 16-row tiles of the activation on fp32 MFMA (16x16x4), whatever the adapters are kept in: products
// and sums are fp32 like the projection's tail, and at ranks of 8 to 64 the matrix pipe is not what bounds them. What a tile's
// rows do not share is handled by slot: a tile's distinct slots are found with wave ballots (a prompt's tile has one or two, a
// decode step's up to 16), each is multiplied with the whole tile, and its results go to its own rows only, by selection and
// not by a zero factor, so that infinities in one request's adapter stay out of the others' rows.
#include <type_traits>

#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

// Four or eight consecutive adapter values at byte `off` of a resource, widened to fp32 (exact).
template <int kType>
__device__ __forceinline__ void load_values(__amdgpu_buffer_rsrc_t r, uint32_t off, f32x4& v) {
    if constexpr (kType == kAdapterF32) {
        v = __builtin_bit_cast(f32x4, ld4(r, off));
    } else {
        const u32x2 raw = ld2(r, off);
        const uint32_t lo = raw.x, hi = raw.y;
        if constexpr (kType == kAdapterF16)
            v = f32x4{half_lo(lo), half_hi(lo), half_lo(hi), half_hi(hi)};
        else
            v = f32x4{as_float(lo << 16), as_float(lo & 0xffff0000u), as_float(hi << 16), as_float(hi & 0xffff0000u)};
    }
}

template <int kType>
struct Raw8 {
    u32x4 v[kType == kAdapterF32 ? 2 : 1];
};
template <int kType>
__device__ __forceinline__ Raw8<kType> load_raw8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    Raw8<kType> x;
    x.v[0] = ld4(r, off);
    if constexpr (kType == kAdapterF32) x.v[1] = ld4(r, off + 16);
    return x;
}
template <int kType>
__device__ __forceinline__ void widen8(const Raw8<kType>& x, float (&f)[8]) {
    const uint32_t w[4] = {x.v[0].x, x.v[0].y, x.v[0].z, x.v[0].w};
    if constexpr (kType == kAdapterF32) {
        const uint32_t u[4] = {x.v[1].x, x.v[1].y, x.v[1].z, x.v[1].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[i] = as_float(w[i]);
            f[4 + i] = as_float(u[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = kType == kAdapterF16 ? half_lo(w[i]) : as_float(w[i] << 16);
            f[2 * i + 1] = kType == kAdapterF16 ? half_hi(w[i]) : as_float(w[i] & 0xffff0000u);
        }
    }
}

constexpr int kElem(int type) { return type == kAdapterF32 ? 4 : 2; }

// The slots of a tile's 16 rows, row m0 + (lane & 15) in each of a wave's four 16-lane groups; -1 for a row without an adapter
// (past the rows, no such slot, nothing loaded there).
__device__ __forceinline__ int tile_slots(const AdapterJob& j, const int* row_slots, int m0, int rows) {
    const int m = m0 + (int)(threadIdx.x & 15);
    const int s = m < rows ? row_slots[m] : -1;
    return s >= 0 && s < j.slots && j.info[s].rank > 0 ? s : -1;
}

// Calls f(slot, rows) for the tile's distinct slots number first, first + step, ...: wave-uniform, `rows` with a bit for each
// of the tile's rows that have the slot.
template <class F>
__device__ __forceinline__ void for_slots(int slot, int first, int step, F f) {
    uint32_t left = (uint32_t)__ballot(slot >= 0) & 0xffffu;
    for (int u = 0; left; u++) {
        const int s = __builtin_amdgcn_readlane(slot, __builtin_ctz(left));
        const uint32_t mine = (uint32_t)__ballot(slot == s) & 0xffffu;
        left &= ~mine;
        if (u >= first && (u - first) % step == 0) f(s, mine);
    }
}

// A_s x for one 16-row tile, kNT tiles of 16 ranks and a share of the inputs: grid ((row tile, distinct slot), (job, rank group),
// input share). The waves of a workgroup divide the share, 32 inputs a step (a lane of an operand holds eight consecutive ones,
// which the eight MFMAs of a step take in turn, so every load is 16 bytes), and add their sums in LDS; the shares of several
// workgroups stay apart in the scratch planes and the expanding kernel adds them, in order.
constexpr int kShrinkWaves = 8;
template <int kType, int kNT>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink_kernel(const AdapterArgs a) {
    __shared__ f32x4 red[kShrinkWaves][kNT][64];
    const int groups = (a.low_stride + 16 * kNT - 1) / (16 * kNT);
    const AdapterJob j = a.job[blockIdx.y / groups];
    const int r0 = (int)(blockIdx.y % groups) * 16 * kNT;
    const int m0 = (int)(blockIdx.x / a.slot_ways) * 16;
    const int wave = wave_id(), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int chunks = a.in / 32;
    const int each = (chunks + kShrinkWaves * a.shares - 1) / (kShrinkWaves * a.shares);
    const int c0 = ((int)blockIdx.z * kShrinkWaves + wave) * each, c1 = min(c0 + each, chunks);
    const __amdgpu_buffer_rsrc_t xr =
        make_rsrc(a.x + (int64_t)m0 * a.in, (uint32_t)min(16, a.rows - m0) * (uint32_t)a.in * 4u);
    const int slot = tile_slots(j, a.row_slots, m0, a.rows);
    for_slots(slot, (int)blockIdx.x % a.slot_ways, a.slot_ways, [&](int s, uint32_t mine) {
        const int rank = j.info[s].rank;
        if (r0 >= rank) return;  // the same for every wave of the workgroup
        const __amdgpu_buffer_rsrc_t ar = make_rsrc(static_cast<const char*>(j.a) + (int64_t)s * j.max_rank * a.in * kElem(kType),
                                                    (uint32_t)rank * (uint32_t)a.in * kElem(kType));
        // rows of other slots are not fetched (an offset past the resource reads zeros)
        const uint32_t x0 = mine >> l16 & 1 ? (uint32_t)l16 * (uint32_t)a.in * 4u + (uint32_t)g * 32u : 0xf0000000u;
        const uint32_t a0 = (uint32_t)(r0 + l16) * (uint32_t)a.in * kElem(kType) + (uint32_t)g * 8u * kElem(kType);
        f32x4 acc[kNT];
#pragma unroll
        for (int t = 0; t < kNT; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int kAhead = kNT == 4 ? 2 : 4;  // steps whose loads go out together
        for (int c = c0; c < c1; c += kAhead) {
            u32x4 xv[kAhead][2];
            Raw8<kType> av[kAhead][kNT];
#pragma unroll
            for (int p = 0; p < kAhead; p++) {
                // past the share: offsets past the resources, zeros (ovfq_adapters_create keeps a slot below 2^30 bytes)
                const bool live = c + p < c1;
                const uint32_t ka = live ? (uint32_t)(c + p) * 32u * kElem(kType) : 0x80000000u;
                const uint32_t kx = live ? (uint32_t)(c + p) * 128u : 0x80000000u;
#pragma unroll
                for (int t = 0; t < kNT; t++)
                    av[p][t] = load_raw8<kType>(ar, a0 + ka + (uint32_t)t * 16u * (uint32_t)a.in * kElem(kType));
                xv[p][0] = ld4(xr, x0 + kx);
                xv[p][1] = ld4(xr, x0 + kx + 16u);
            }
#pragma unroll
            for (int p = 0; p < kAhead; p++) {
                const float x[8] = {as_float(xv[p][0].x), as_float(xv[p][0].y), as_float(xv[p][0].z), as_float(xv[p][0].w),
                                    as_float(xv[p][1].x), as_float(xv[p][1].y), as_float(xv[p][1].z), as_float(xv[p][1].w)};
#pragma unroll
                for (int t = 0; t < kNT; t++) {
                    float w[8];
                    widen8<kType>(av[p][t], w);
#pragma unroll
                    for (int i = 0; i < 8; i++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], w[i], acc[t], 0, 0, 0);
                }
            }
        }
        __syncthreads();  // the last slot's sums have been read
#pragma unroll
        for (int t = 0; t < kNT; t++) red[wave][t][lane] = acc[t];
        __syncthreads();
        for (int t = wave; t < kNT; t += kShrinkWaves) {
            f32x4 v = red[0][t][lane];
#pragma unroll
            for (int w = 1; w < kShrinkWaves; w++) v += red[w][t][lane];
            // lane (g, l16) holds rows 4 g .. 4 g + 3 of rank r0 + 16 t + l16
            const int r = r0 + 16 * t + l16;
            float* low = j.low + ((int64_t)blockIdx.z * a.rows + m0 + 4 * g) * a.low_stride + r;
            if (r < a.low_stride) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (mine >> (4 * g + i) & 1) low[(int64_t)i * a.low_stride] = v[i];
            }
        }
    });
}

// The products of one slot for a 16-row tile and kT tiles of 16 outputs: acc[t] (lane (g, l16): rows 4 g .. 4 g + 3, output
// n0 + 16 t + l16) = sum_r low[m][r] B[n][r], 16 ranks a step.
template <int kType, int kT>
__device__ __forceinline__ void expand_slot(const AdapterArgs& a, const AdapterJob& j, int s, int m0, int n0, f32x4 (&acc)[kT]) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int pad = rank_pad(j.info[s].rank);
    const __amdgpu_buffer_rsrc_t br =
        make_rsrc(static_cast<const char*>(j.b) + (int64_t)s * j.out * j.b_stride * kElem(kType),
                  (uint32_t)j.out * (uint32_t)pad * kElem(kType));
    const int left = min(16, a.rows - m0);
#pragma unroll
    for (int t = 0; t < kT; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int r = 0; r < pad; r += 16) {
        const int at = r + 4 * g;  // this lane's four ranks
        f32x4 b[kT], low = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < kT; t++) {
            const uint32_t off = (uint32_t)(n0 + 16 * t + l16) * (uint32_t)pad * kElem(kType) + (uint32_t)at * kElem(kType);
            load_values<kType>(br, at < pad && n0 + 16 * t + l16 < j.out ? off : 0xf0000000u, b[t]);
        }
        for (int sh = 0; sh < a.shares; sh++) {
            const __amdgpu_buffer_rsrc_t lr = make_rsrc(j.low + ((int64_t)sh * a.rows + m0) * a.low_stride,
                                                        (uint32_t)left * (uint32_t)a.low_stride * 4u);
            low += __builtin_bit_cast(f32x4, ld4(lr, at < pad ? (uint32_t)(l16 * a.low_stride + at) * 4u : 0xf0000000u));
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < kT; t++) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(low[i], b[t][i], acc[t], 0, 0, 0);
    }
}

// grid (row tiles, output tiles, jobs): a wave per 16 rows x 64 outputs.
template <int kType>
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterArgs a) {
    constexpr int kT = 4;
    const AdapterJob j = a.job[blockIdx.z];
    const int m0 = (int)blockIdx.x * 16, n0 = ((int)blockIdx.y * 4 + wave_id()) * 16 * kT;
    if (n0 >= j.out) return;
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int slot = tile_slots(j, a.row_slots, m0, a.rows);
    const uint32_t any = (uint32_t)__ballot(slot >= 0) & 0xffffu;
    if (!any) return;
    f32x4 y[kT];
    float* yp = j.y + (int64_t)(m0 + 4 * g) * j.out + n0 + l16;
#pragma unroll
    for (int t = 0; t < kT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (any >> (4 * g + i) & 1 && n0 + 16 * t + l16 < j.out) y[t][i] = yp[(int64_t)i * j.out + 16 * t];
    for_slots(slot, 0, 1, [&](int s, uint32_t mine) {
        f32x4 acc[kT];
        expand_slot<kType, kT>(a, j, s, m0, n0, acc);
        const float scale = j.info[s].scale;
#pragma unroll
        for (int t = 0; t < kT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (mine >> (4 * g + i) & 1) y[t][i] = fmaf(acc[t][i], scale, y[t][i]);
    });
#pragma unroll
    for (int t = 0; t < kT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (any >> (4 * g + i) & 1 && n0 + 16 * t + l16 < j.out) yp[(int64_t)i * j.out + 16 * t] = y[t][i];
}

__global__ __launch_bounds__(256) void adapter_slot_kernel(AdapterSlot* info, int first, int count, int rank, float scale) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i < count) info[first + i] = AdapterSlot{rank, scale};
}

// B [out][rank] -> rows of rank_pad(rank) values, zeros past the rank. T: the values' storage width.
template <class T>
__global__ __launch_bounds__(256) void adapter_pad_kernel(const T* __restrict__ src, T* __restrict__ dst, int64_t n, int rank,
                                                          int pad) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t row = i / pad;
    const int r = (int)(i - row * pad);
    dst[i] = r < rank ? src[row * rank + r] : T(0);
}

template <int kType>
hipError_t launch_apply(const AdapterArgs& a, int jobs, hipStream_t st) {
    int out = 0;
    for (int i = 0; i < jobs; i++) out = a.job[i].out > out ? a.job[i].out : out;
    const unsigned tiles = (unsigned)((a.rows + 15) / 16);
    const auto shrink = [&](auto nt) {
        constexpr int kNT = decltype(nt)::value;
        const unsigned groups = (unsigned)((a.low_stride + 16 * kNT - 1) / (16 * kNT));
        hipLaunchKernelGGL((adapter_shrink_kernel<kType, kNT>), dim3(tiles * (unsigned)a.slot_ways, (unsigned)jobs * groups, (unsigned)a.shares),
                           dim3(64 * kShrinkWaves), 0, st, a);
    };
    if (a.rows <= 64 || a.low_stride <= 16)
        shrink(std::integral_constant<int, 1>{});
    else if (a.low_stride <= 32)
        shrink(std::integral_constant<int, 2>{});
    else
        shrink(std::integral_constant<int, 4>{});
    hipLaunchKernelGGL(adapter_expand_kernel<kType>, dim3(tiles, (unsigned)((out + 255) / 256), (unsigned)jobs), dim3(256), 0, st,
                       a);
    return hipGetLastError();
}

}  // namespace

void plan_adapters(AdapterArgs& a, int jobs, int max_rank) {
    a.low_stride = (max_rank + 15) & ~15;
    const int tiles = (a.rows + 15) / 16;
    const int nt = a.rows <= 64 || a.low_stride <= 16 ? 1 : a.low_stride <= 32 ? 2 : 4;
    const int wgs = tiles * jobs * ((a.low_stride + 16 * nt - 1) / (16 * nt));
    const int most = (a.in / 32 + 4 * kShrinkWaves - 1) / (4 * kShrinkWaves);  // four steps a wave at least
    a.shares = (256 + wgs - 1) / wgs;
    if (a.shares > most) a.shares = most;
    int slots = 1;
    for (int i = 0; i < jobs; i++) slots = a.job[i].slots > slots ? a.job[i].slots : slots;
    a.slot_ways = a.rows > 64 ? 2 : a.rows < 16 ? a.rows : 16;
    if (a.slot_ways > slots) a.slot_ways = slots;
}

hipError_t launch_adapters(const AdapterArgs& a, int type, int jobs, hipStream_t st) {
    if (type == kAdapterF32) return launch_apply<kAdapterF32>(a, jobs, st);
    if (type == kAdapterF16) return launch_apply<kAdapterF16>(a, jobs, st);
    return launch_apply<kAdapterBF16>(a, jobs, st);
}

hipError_t launch_adapter_slots(AdapterSlot* info, int first, int count, int rank, float scale, hipStream_t st) {
    hipLaunchKernelGGL(adapter_slot_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, st, info, first, count, rank,
                       scale);
    return hipGetLastError();
}

hipError_t launch_adapter_pad(const void* src, void* dst, int out, int rank, int elem, hipStream_t st) {
    const int pad = rank_pad(rank);
    const int64_t n = (int64_t)out * pad;
    const dim3 grid((unsigned)((n + 255) / 256));
    if (elem == 4)
        hipLaunchKernelGGL(adapter_pad_kernel<uint32_t>, grid, dim3(256), 0, st, (const uint32_t*)src, (uint32_t*)dst, n, rank,
                           pad);
    else
        hipLaunchKernelGGL(adapter_pad_kernel<uint16_t>, grid, dim3(256), 0, st, (const uint16_t*)src, (uint16_t*)dst, n, rank,
                           pad);
    return hipGetLastError();
}

}  // namespace ovfq
