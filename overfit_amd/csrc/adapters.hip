// adapters.hip — low-rank adapters of many requests beside a shared projection: for every activation row m with an adapter
// slot s, y[m] += scale_s * B_s (A_s x[m]), A_s [rank][in], B_s [out][rank].
//
// Two steps: the rows' products A_s x[m] into scratch planes (shrink), in one launch with the quantisation of the activation
// where the projection has one, then B_s times them (expand), in the epilogue of the projection kernels that take adapters and
// in a launch of its own behind the others (adapter_tile.h). Products and sums are fp32 like the projection's tail, whatever the
// adapters are kept in.
#include <type_traits>

#include "act_quant.h"
#include "adapter_tile.h"
#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

// fp32 operands of bf16 MFMA: a value is the sum of three bf16 parts (8 significant bits each, cut off, so every part and rest is
// exact), and the products of parts are exact in fp32. Eight consecutive values of a lane, two to a dword.
struct Parts {
    u32x4 part[3];
};
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
__device__ __forceinline__ float cut(float v) { return as_float(__builtin_bit_cast(uint32_t, v) & 0xffff0000u); }
template <int kParts>
__device__ __forceinline__ void split_pair(float v0, float v1, int i, u32x4 (&part)[3]) {
    part[0][i] = upper_halves(v0, v1);
    const float r0 = v0 - cut(v0), r1 = v1 - cut(v1);
    part[1][i] = upper_halves(r0, r1);
    if constexpr (kParts == 3) part[2][i] = upper_halves(r0 - cut(r0), r1 - cut(r1));
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A lane's eight values of a piece of A, at byte `off` of the resource.
template <int kType>
struct Raw8 {
    u32x4 v[kType == kAdapterF32 ? 2 : 1];
};
template <int kType>
__device__ __forceinline__ Raw8<kType> load_raw8(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    Raw8<kType> x;
    x.v[0] = ld4(r, off);
    if constexpr (kType == kAdapterF32) x.v[1] = ld4(r, off + 1024);
    return x;
}

// acc += x w over 32 inputs, the small products first. bf16 adapters are their own part (three MFMAs), fp16 ones (11 bits)
// two parts (six, every product exact), fp32 ones three: of their nine products the three that are 2^-24 of the whole or less are
// left out. (An infinity's parts are itself and NaN, so its products are NaN.)
template <int kType>
__device__ __forceinline__ f32x4 multiply(const Parts& x, const Raw8<kType>& w, f32x4 acc) {
    if constexpr (kType == kAdapterBF16) {
#pragma unroll
        for (int p = 2; p >= 0; p--) acc = mfma_bf16(x.part[p], w.v[0], acc);
    } else {
        u32x4 part[3];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (kType == kAdapterF16) {
                const uint32_t u = w.v[0][i];
                split_pair<2>(half_lo(u), half_hi(u), i, part);
            } else {
                const uint32_t u0 = w.v[i >> 1][2 * (i & 1)], u1 = w.v[i >> 1][2 * (i & 1) + 1];
                split_pair<3>(as_float(u0), as_float(u1), i, part);
            }
        }
        if constexpr (kType == kAdapterF16) {
#pragma unroll
            for (int p = 2; p >= 0; p--) acc = mfma_bf16(x.part[p], part[1], acc);
#pragma unroll
            for (int p = 2; p >= 0; p--) acc = mfma_bf16(x.part[p], part[0], acc);
        } else {
            acc = mfma_bf16(x.part[2], part[0], acc);
            acc = mfma_bf16(x.part[0], part[2], acc);
            acc = mfma_bf16(x.part[1], part[1], acc);
            acc = mfma_bf16(x.part[1], part[0], acc);
            acc = mfma_bf16(x.part[0], part[1], acc);
            acc = mfma_bf16(x.part[0], part[0], acc);
        }
    }
    return acc;
}

// A_s x for one 16-row tile, kNV rank tiles (16 ranks of one of the jobs each; two jobs share the loads of x) and a share of
// the inputs: grid (way of the tile's distinct slots + ways * row tile, rank tile group + groups * share). Its waves divide the
// share, 128 inputs a round, and add their sums in LDS; the shares of several workgroups stay apart in the scratch planes and are
// added, in order, where they are used. Rows of the grid after these quantise the activation.
//
// Bound by latencies: the slots, then A and x, then the sums, behind a launch of 3 to 4.5 us. Three things were taken out of that
// chain (18.7 us at 331 rows of q/k/v and rank 32, of which the products were less than one). Operands loaded where they lie, a
// lane's 16 or 32 bytes of its own row, are 64 pieces an instruction: A is kept in operand order, and x goes through LDS, two
// rows' 512 bytes an instruction in, a lane's own 32 bytes out. A slot's rank, another dependent load, is waited for before A
// only past the first 16 ranks. And the workgroup's place comes from the grid and from the host, not from divisions.
constexpr int kShrinkWaves = 4, kRound = 128, kXRow = kRound + 4;
template <int kType, int kNV>
__global__ __launch_bounds__(64 * kShrinkWaves, 3) void adapter_shrink_kernel(const AdapterArgs a, const ActQuantJob quant) {
    const int shrink_rows = a.groups * a.shares;
    if ((int)blockIdx.y >= shrink_rows) {
        quantize_part(quant, (int64_t)((int)blockIdx.y - shrink_rows) * gridDim.x + blockIdx.x);
        return;
    }
    if ((int)blockIdx.x >= a.shrink_x) return;
    // x of the waves' rounds; their sums afterwards
    __shared__ __align__(16) float lds[kShrinkWaves][16 * kXRow];
    static_assert(kNV * 256 <= 16 * kXRow, "sums of a wave");
    const int per_job = a.low_stride / 16;
    int v0 = (int)blockIdx.y, share = 0;
    while (v0 >= a.groups) {
        v0 -= a.groups;
        share++;
    }
    v0 *= kNV;
    const int m0 = ((int)blockIdx.x >> a.way_shift) * 16, way = (int)blockIdx.x & ((1 << a.way_shift) - 1);
    const int wave = wave_id(), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int m = m0 + l16;
    const int slot = m < a.rows ? a.row_slots[m] : -1;  // of row m0 + l16 in each 16-lane group
    const int c0 = (share * kShrinkWaves + wave) * a.each, c1 = min(c0 + a.each, a.in / 32);
    const __amdgpu_buffer_rsrc_t xr =
        make_rsrc(a.x + (int64_t)m0 * a.in, (uint32_t)min(16, a.rows - m0) * (uint32_t)a.in * 4u);
    struct Tile {
        const char* a;
        const AdapterSlot* info;
        float* low;
        AdapterRow* row;
        int slots, max_rank, r0;
    } tl[kNV];
    bool first_ranks = false;
#pragma unroll
    for (int t = 0; t < kNV; t++) {
        int job = 0, r = v0 + t;
        while (r >= per_job) {
            r -= per_job;
            job++;
        }
        const AdapterJob j = adapter_job(a, job < a.jobs ? job : 0);
        tl[t] = Tile{static_cast<const char*>(j.a), j.info, j.low, j.row, job < a.jobs ? j.slots : 0, j.max_rank, r * 16};
        first_ranks = first_ranks || (tl[t].slots && !r);
    }
    // What the rows have of the sets; this workgroup writes it down for the kernels that expand if it is the first of its rows.
    AdapterSlot info[kNV];
#pragma unroll
    for (int t = 0; t < kNV; t++) info[t] = slot >= 0 && slot < tl[t].slots ? tl[t].info[slot] : AdapterSlot{0, 0.0f};
    uint32_t left = (uint32_t)__ballot(slot >= 0) & 0xffffu;
    float* xs = lds[wave];
    for (int u = 0; left; u++) {
        const int first = __builtin_ctz(left);
        const int s = __builtin_amdgcn_readlane(slot, first);
        const uint32_t mine = (uint32_t)__ballot(slot == s) & 0xffffu;
        left &= ~mine;
        if ((u & ((1 << a.way_shift) - 1)) != way) continue;
        // (the same for every wave of the workgroup)
        if (!first_ranks) {
            bool any = false;
#pragma unroll
            for (int t = 0; t < kNV; t++) any = any || tl[t].r0 < __builtin_amdgcn_readlane(info[t].rank, first);
            if (!any) continue;
        }
        constexpr uint32_t kAbsent = 0xf0000000u;  // past every resource: reads zeros
        __amdgpu_buffer_rsrc_t ar[kNV];
#pragma unroll
        for (int t = 0; t < kNV; t++) {
            const bool in = s < tl[t].slots && tl[t].r0 < tl[t].max_rank;
            const int64_t size = adapter_a_slot(a.in, tl[t].max_rank) * adapter_elem(kType);
            ar[t] = make_rsrc(tl[t].a + (in ? s * size + (int64_t)tl[t].r0 * a.in * adapter_elem(kType) : 0),
                              in ? 16u * (uint32_t)a.in * adapter_elem(kType) : 0u);
        }
        f32x4 acc[kNV];
#pragma unroll
        for (int t = 0; t < kNV; t++) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        u32x4 xv[8];
        Raw8<kType> av[4][kNV];
        auto load_a = [&](int c, int p) {
#pragma unroll
            for (int t = 0; t < kNV; t++)
                av[p][t] = load_raw8<kType>(ar[t], c + p < c1 ? (uint32_t)(c + p) * (512u * adapter_elem(kType)) + 16u * (uint32_t)lane
                                                              : kAbsent);
        };
        auto load_x = [&](int c) {  // rows of other slots are not fetched
            const int k = c * 32 + 4 * (lane & 31);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = 2 * i + (lane >> 5);
                xv[i] = ld4(xr, (mine >> r & 1) && k < c1 * 32 ? ((uint32_t)r * (uint32_t)a.in + (uint32_t)k) * 4u : kAbsent);
            }
        };
        load_x(c0);
#pragma unroll
        for (int p = 0; p < 4; p++) load_a(c0, p);
        __syncthreads();  // the last slot's sums have been read
        for (int c = c0; c < c1; c += 4) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                *reinterpret_cast<u32x4*>(xs + (2 * i + (lane >> 5)) * kXRow + 4 * (lane & 31)) = xv[i];
            wave_sync();
            const bool more = c + 4 < c1;
            if (more) load_x(c + 4);
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(xs + l16 * kXRow + 32 * p + 8 * g);
                const f32x4 hi = *reinterpret_cast<const f32x4*>(xs + l16 * kXRow + 32 * p + 8 * g + 4);
                Parts x;
                split_pair<3>(lo[0], lo[1], 0, x.part);
                split_pair<3>(lo[2], lo[3], 1, x.part);
                split_pair<3>(hi[0], hi[1], 2, x.part);
                split_pair<3>(hi[2], hi[3], 3, x.part);
#pragma unroll
                for (int t = 0; t < kNV; t++) acc[t] = multiply<kType>(x, av[p][t], acc[t]);
                if (more) load_a(c + 4, p);
            }
            wave_sync();
        }
        // (the wave's own words: its x is used up)
#pragma unroll
        for (int t = 0; t < kNV; t++) *reinterpret_cast<f32x4*>(xs + t * 256 + 4 * lane) = acc[t];
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kNV; t++) {
            if (wave != t || tl[t].r0 >= __builtin_amdgcn_readlane(info[t].rank, first)) continue;
            f32x4 v = *reinterpret_cast<const f32x4*>(lds[0] + t * 256 + 4 * lane);
#pragma unroll
            for (int w = 1; w < kShrinkWaves; w++) v += *reinterpret_cast<const f32x4*>(lds[w] + t * 256 + 4 * lane);
            // lane (g, l16) holds rows 4 g .. 4 g + 3 of rank r0 + l16
            float* low = tl[t].low + ((int64_t)share * a.rows + m0 + 4 * g) * a.low_stride + tl[t].r0 + l16;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (mine >> (4 * g + i) & 1) low[(int64_t)i * a.low_stride] = v[i];
        }
    }
#pragma unroll
    for (int t = 0; t < kNV; t++)
        if (tl[t].slots && !tl[t].r0 && !share && !way && wave == kShrinkWaves - 1 - t && lane < 16 && m < a.rows)
            tl[t].row[m] = AdapterRow{info[t].rank > 0 ? (uint32_t)slot << 16 | (uint32_t)rank_pad(info[t].rank) : 0u, info[t].scale};
}

// Outputs that a projection kernel without adapters has written, or the tiles of many slots that one has left: 4 rows x 256 outputs a
// workgroup, an output a thread, with 16 ranks of the rows' B at a time. A row's slot is the same for the whole wave, so that B
// takes scalar resources and one offset a row; the low-rank products are LDS broadcasts. Bound by B, which every row reads from L2:
// grid (8 * groups of rows, groups of 8 output tiles, jobs), the rows of an output tile on one XCD (gate/up of 14336, 256 rows over
// 32 slots of rank 16: 40 us, 55 with the tiles over MFMA layouts and per-lane addresses).
constexpr int kExpandRows = 4;
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterArgs a) {
    constexpr int kRow = 256 + 4;
    const AdapterJob j = adapter_job(a, (int)blockIdx.z);
    __shared__ __align__(16) float low[kExpandRows * kRow];
    const int m0 = ((int)blockIdx.x >> 3) * kExpandRows, o_tile = (int)blockIdx.y * 8 + ((int)blockIdx.x & 7);
    if (!j.slots || o_tile * 256 >= j.out) return;
    const int l0 = m0 & 15;
    const AdapterRow row = adapter_row(a, j, m0 - l0 + (int)(threadIdx.x & 15));  // of the rows' tile of 16
    if (a.by_row && !adapter_many(row.key, a.by_row)) return;  // the whole workgroup
    if (!((uint32_t)__ballot(row.pad() != 0) >> l0 & ((1u << kExpandRows) - 1))) return;
    // the products, their shares added
    const int quads = a.low_stride / 4;
    if (const int m = wave_id(); m0 + m < a.rows)
        for (int q = (int)threadIdx.x & 63; q < quads; q += 64) {
            f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
            for (int s0 = 0; s0 < a.shares; s0 += 4) {
                f32x4 v[4];
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const int64_t share = s0 + s < a.shares ? s0 + s : 0;
                    v[s] = *reinterpret_cast<const f32x4*>(j.low + (share * a.rows + m0 + m) * a.low_stride + 4 * q);
                }
#pragma unroll
                for (int s = 0; s < 4; s++)
                    if (s0 + s < a.shares) sum += v[s];
            }
            *reinterpret_cast<f32x4*>(low + m * kRow + 4 * q) = sum;
        }
    const int n = o_tile * 256 + (int)threadIdx.x;
    const int elem = adapter_elem(a.type);
    int pad[kExpandRows], most = 0;
    float scale[kExpandRows], y[kExpandRows], sum[kExpandRows];
    __amdgpu_buffer_rsrc_t br[kExpandRows];
    uint32_t at[kExpandRows];
#pragma unroll
    for (int i = 0; i < kExpandRows; i++) {
        const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)row.key, l0 + i);
        pad[i] = (int)(key & 0xffffu);  // 0 past the rows
        most = max(most, pad[i]);
        scale[i] = as_float((uint32_t)__builtin_amdgcn_readlane((int)__builtin_bit_cast(uint32_t, row.scale), l0 + i));
        const int steps = adapter_tiles16(pad[i]);
        br[i] = make_rsrc(adapter_b(a, j, pad[i] ? (int)(key >> 16) : 0), (uint32_t)(adapter_tiles16(j.out) * steps * 256 * elem));
        at[i] = adapter_b_at(n, 0, steps) * (uint32_t)elem;
        if (pad[i] && n < j.out) y[i] = j.y[(int64_t)(m0 + i) * j.out + n];
        sum[i] = 0.0f;
    }
    u32x4 b[kExpandRows][4];
    const auto load = [&](int r0) {
#pragma unroll
        for (int i = 0; i < kExpandRows; i++)
#pragma unroll
            for (int q = 0; q < 4; q++)  // (past the slot's ranks: zeros or other outputs' values, unused)
                b[i][q] = adapter_load4(a.type, br[i], at[i] + (uint32_t)((r0 * 16 + q * 64) * elem));
    };
    load(0);
    __syncthreads();
#pragma unroll 1
    for (int r0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kExpandRows; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (r0 + 4 * q >= pad[i]) continue;
                const f32x4 l = *reinterpret_cast<const f32x4*>(low + i * kRow + r0 + 4 * q);
                const adapter_f32x4 w = adapter_widen4(a.type, b[i][q]);
#pragma unroll
                for (int c = 0; c < 4; c++) sum[i] = fmaf(l[c], w[c], sum[i]);
            }
        r0 += 16;
        if (r0 >= most) break;
        load(r0);
    }
#pragma unroll
    for (int i = 0; i < kExpandRows; i++)
        if (pad[i] && n < j.out) j.y[(int64_t)(m0 + i) * j.out + n] = fmaf(sum[i], scale[i], y[i]);
}

__global__ __launch_bounds__(256) void adapter_slot_kernel(AdapterSlot* info, int first, int count, int rank, float scale) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i < count) info[first + i] = AdapterSlot{rank, scale};
}

// A and B into operand order; T: the values' storage width. A: values i = ((tile, chunk, half), lane, e), E = 16 / sizeof(T) values
// a lane and half; B: ((output tile, rank step), lane, four ranks).
template <class T>
__global__ __launch_bounds__(256) void adapter_pack_kernel(const T* __restrict__ a, const T* __restrict__ b, T* __restrict__ pa,
                                                           T* __restrict__ pb, int in, int out, int rank) {
    constexpr int E = 16 / sizeof(T), kHalves = 8 / E;
    const int steps = adapter_tiles16(rank);
    const int64_t na = (int64_t)steps * 16 * in, nb = (int64_t)adapter_tiles16(out) * steps * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < na + nb; i += (int64_t)gridDim.x * 256) {
        if (i < na) {
            const int e = (int)(i % E), lane = (int)(i / E % 64);
            const int64_t piece = i / (E * 64);
            const int half = (int)(piece % kHalves), c = (int)(piece / kHalves % (in / 32)), t = (int)(piece / kHalves / (in / 32));
            const int r = 16 * t + (lane & 15), k = 32 * c + 8 * (lane >> 4) + E * half + e;
            pa[i] = r < rank ? a[(int64_t)r * in + k] : T(0);
        } else {
            const int64_t q = i - na;
            const int e = (int)(q & 3), lane = (int)(q >> 2 & 63);
            const int64_t piece = q >> 8;
            const int64_t n = piece / steps * 16 + (lane & 15);
            const int r = (int)(piece % steps) * 16 + 4 * (lane >> 4) + e;
            pb[q] = r < rank && n < out ? b[n * rank + r] : T(0);
        }
    }
}

template <int kType>
hipError_t launch_shrink(const AdapterArgs& a, const ActQuantJob& quant, hipStream_t st) {
    // quantising parts fill rows of their own behind the others, at least 64 workgroups wide
    const int64_t parts = quant.parts(), want = parts < 64 ? parts : 64, least = a.shrink_x > want ? a.shrink_x : want;
    // Consecutive workgroups go to the 8 XCDs in turn. Many row tiles: a multiple of 8, so that a tile's workgroups run on one XCD
    // and share its L2's copy of x; few: an odd number, so that they spread over all.
    const int64_t x = a.rows > 64 ? (least + 7) / 8 * 8 : least | 1;
    const dim3 grid((unsigned)x, (unsigned)(a.groups * a.shares + (parts + x - 1) / x)), wg(64 * kShrinkWaves);
    if (a.rank_tiles == 1)
        hipLaunchKernelGGL((adapter_shrink_kernel<kType, 1>), grid, wg, 0, st, a, quant);
    else
        hipLaunchKernelGGL((adapter_shrink_kernel<kType, 2>), grid, wg, 0, st, a, quant);
    return hipGetLastError();
}

}  // namespace

void plan_adapters(AdapterArgs& a, int max_rank) {
    a.low_stride = (max_rank + 15) & ~15;
    int slots = 1;
    for (int i = 0; i < a.jobs; i++) slots = a.job[i].slots > slots ? a.job[i].slots : slots;
    const int tiles = (a.rows + 15) / 16, all = a.jobs * (a.low_stride / 16);
    const int kMostShares = a.rows <= 32 ? 8 : 4;
    // two rank tiles beside each other where that leaves 128 workgroups
    a.rank_tiles = all > 1 && tiles * ((all + 1) / 2) * kMostShares >= 128 ? 2 : 1;
    a.groups = (all + a.rank_tiles - 1) / a.rank_tiles;
    const int wgs = tiles * a.groups;
    const int most = (a.in / 32 + 4 * kShrinkWaves - 1) / (4 * kShrinkWaves);  // a round a wave at least
    a.shares = (256 + wgs - 1) / wgs;
    if (a.shares > most) a.shares = most;
    if (a.shares > kMostShares) a.shares = kMostShares;
    a.each = (a.in / 32 + kShrinkWaves * a.shares - 1) / (kShrinkWaves * a.shares);
    // A workgroup for each of a tile's slots at a few rows, which may all differ. At many, two, for the tiles where one request ends
    // and the next begins; four with one rank tile and sets of more slots than the projections take in turn (us, two / four / eight:
    // gate/up of 14336 at 256 rows, every row its own of 32 slots 27.4 / 16.3 / 17.2, three requests 7.7 / 7.7 / 12.1; down 14336 ->
    // 4096 at 300 rows 67.4 / 41.0 / 27.5, 14.1 / 16.1 / 20.9; with two rank tiles, q/k/v of 4096 at 400 rows 33.0 / 33.4 / 29.8, 9.9 / 16.1 /
    // 18.9: workgroups without a slot wait for a place all the same).
    a.way_shift = 0;
    const int ways = a.rows <= 64 ? 4 : a.rank_tiles == 1 && slots > kAdapterFew ? 2 : 1;
    while (a.way_shift < ways && 1 << a.way_shift < slots && 1 << a.way_shift < a.rows) a.way_shift++;
    a.shrink_x = tiles << a.way_shift;
}

hipError_t launch_adapters_shrink(const AdapterArgs& a, const ActQuantJob& quant, hipStream_t st) {
    if (a.type == kAdapterF32) return launch_shrink<kAdapterF32>(a, quant, st);
    if (a.type == kAdapterF16) return launch_shrink<kAdapterF16>(a, quant, st);
    return launch_shrink<kAdapterBF16>(a, quant, st);
}

hipError_t launch_adapters_expand(const AdapterArgs& a, hipStream_t st) {
    int out = 0;
    for (int i = 0; i < a.jobs; i++) out = a.job[i].slots && a.job[i].out > out ? a.job[i].out : out;
    hipLaunchKernelGGL(adapter_expand_kernel, dim3((unsigned)((a.rows + kExpandRows - 1) / kExpandRows * 8), (unsigned)((out + 2047) / 2048),
                                                      (unsigned)a.jobs),
                       dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_adapter_slots(AdapterSlot* info, int first, int count, int rank, float scale, hipStream_t st) {
    hipLaunchKernelGGL(adapter_slot_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, st, info, first, count, rank,
                       scale);
    return hipGetLastError();
}

hipError_t launch_adapter_pack(const void* a, const void* b, void* a_slot, void* b_slot, int type, int in, int out, int rank,
                               hipStream_t st) {
    const int64_t n = adapter_a_slot(in, rank) + adapter_b_slot(out, rank);
    const dim3 grid((unsigned)((n + 1023) / 1024 < 4096 ? (n + 1023) / 1024 : 4096));
    if (type == kAdapterF32)
        hipLaunchKernelGGL(adapter_pack_kernel<uint32_t>, grid, dim3(256), 0, st, (const uint32_t*)a, (const uint32_t*)b,
                           (uint32_t*)a_slot, (uint32_t*)b_slot, in, out, rank);
    else
        hipLaunchKernelGGL(adapter_pack_kernel<uint16_t>, grid, dim3(256), 0, st, (const uint16_t*)a, (const uint16_t*)b,
                           (uint16_t*)a_slot, (uint16_t*)b_slot, in, out, rank);
    return hipGetLastError();
}

}  // namespace ovfq
