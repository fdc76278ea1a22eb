// adapter_tile.h — B times the rows' low-rank products, for the epilogues of the projection kernels and for the launch that
// adds adapters to finished outputs (adapters.hip). Products and sums are fp32 whatever the adapters are kept in.
//
// Rows share a multiplication only where they share the slot. Tiles of one or two slots (a prompt's) go over fp32 MFMA
// (16x16x4): each slot is multiplied with the whole tile and its results go to its own rows only, by selection and not by a
// zero factor, so that an infinity in one request's adapter stays out of the others' rows. Tiles of more slots (a decode
// step's) go output by output: a lane loads the row of B that its output's slot names, so all loads are in flight at once,
// where a walk over 16 slots waited for each.
#pragma once

#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

struct NoAdapters {};  // a projection kernel's adapter argument where the call has none

typedef float adapter_f32x4 __attribute__((ext_vector_type(4)));

// The adapters of weight i, chosen by select among the kernel's arguments: an index known at run time would read them again
// through memory, two more latencies at the start of a launch.
__device__ __forceinline__ AdapterJob adapter_job(const AdapterArgs& e, int i) {
    AdapterJob j = e.job[0];
#pragma unroll
    for (int k = 1; k < kMaxJobs; k++) {
        const bool take = i == k;
        const AdapterJob& o = e.job[k];
        j.a = take ? o.a : j.a;
        j.b = take ? o.b : j.b;
        j.info = take ? o.info : j.info;
        j.row = take ? o.row : j.row;
        j.low = take ? o.low : j.low;
        j.y = take ? o.y : j.y;
        j.slots = take ? o.slots : j.slots;
        j.max_rank = take ? o.max_rank : j.max_rank;
        j.out = take ? o.out : j.out;
    }
    return j;
}

// Four consecutive adapter values, and their fp32 widening (exact).
__device__ __forceinline__ u32x4 adapter_load4(int type, __amdgpu_buffer_rsrc_t r, uint32_t off) {
    if (type == kAdapterF32) return ld4(r, off);
    const u32x2 v = ld2(r, off);
    return u32x4{v.x, v.y, 0u, 0u};
}
__device__ __forceinline__ adapter_f32x4 adapter_widen4(int type, u32x4 v) {
    const uint32_t a = v.x, b = v.y, c = v.z, d = v.w;
    if (type == kAdapterF32) return adapter_f32x4{as_float(a), as_float(b), as_float(c), as_float(d)};
    if (type == kAdapterF16) return adapter_f32x4{half_lo(a), half_hi(a), half_lo(b), half_hi(b)};
    return adapter_f32x4{as_float(a << 16), as_float(a & 0xffff0000u), as_float(b << 16), as_float(b & 0xffff0000u)};
}

// The adapter of activation row m; pad 0: none (past the rows too).
__device__ __forceinline__ AdapterRow adapter_row(const AdapterArgs& e, const AdapterJob& j, int m) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(j.row, (uint32_t)e.rows * 8u);
    const u32x2 v = ld2(r, (uint32_t)m * 8u);
    const uint32_t scale = v.y;
    return AdapterRow{v.x, as_float(scale)};
}

// The low-rank products of kRows (a multiple of 16) activation rows from m0 on, ranks r0 .. r0 + kRanks, their shares added: into
// LDS rows of kRanks + 4 floats, by the kThreads threads of the workgroup. Rows past the launch's hold zeros. In two steps, so
// that other loads can go out between: every load of the first is in flight at once (four shares at a time).
template <int kRows, int kRanks, int kThreads>
struct AdapterStage {
    static constexpr int kQuads = kRows * kRanks / 4, kPer = (kQuads + kThreads - 1) / kThreads;
    u32x4 v[kPer][4];

    __device__ __forceinline__ static uint32_t offset(const AdapterArgs& e, int i, int r0) {
        const int q = (int)threadIdx.x + kThreads * i, row = q / (kRanks / 4), c = r0 + 4 * (q % (kRanks / 4));
        return q < kQuads && c < e.low_stride ? (uint32_t)(row * e.low_stride + c) * 4u : 0xf0000000u;
    }
    __device__ __forceinline__ void load(const AdapterArgs& e, const AdapterJob& j, int m0, int r0, int sh0 = 0) {
        const int64_t left = e.rows - m0;
        const uint32_t bytes = (uint32_t)(left < kRows ? left : kRows) * (uint32_t)e.low_stride * 4u;
#pragma unroll
        for (int sh = 0; sh < 4; sh++) {
            const __amdgpu_buffer_rsrc_t r =
                make_rsrc(j.low + ((int64_t)(sh0 + sh) * e.rows + m0) * e.low_stride, sh0 + sh < e.shares ? bytes : 0u);
#pragma unroll
            for (int i = 0; i < kPer; i++) v[i][sh] = ld4(r, offset(e, i, r0));
        }
    }
    __device__ __forceinline__ void store(const AdapterArgs& e, const AdapterJob& j, int m0, int r0, float* lds) {
        adapter_f32x4 sum[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) sum[i] = adapter_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int sh0 = 0;;) {
#pragma unroll
            for (int i = 0; i < kPer; i++)
#pragma unroll
                for (int sh = 0; sh < 4; sh++) sum[i] += __builtin_bit_cast(adapter_f32x4, v[i][sh]);
            sh0 += 4;
            if (sh0 >= e.shares) break;
            load(e, j, m0, r0, sh0);
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int q = (int)threadIdx.x + kThreads * i;
            if (q < kQuads) *reinterpret_cast<adapter_f32x4*>(lds + q / (kRanks / 4) * (kRanks + 4) + 4 * (q % (kRanks / 4))) = sum[i];
        }
    }
};

// The workgroup's LDS stores before, its loads after; DMAs into LDS stay in flight.
__device__ __forceinline__ void adapter_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A slot's B, and where ranks r .. r + 3 (r a multiple of 4) of output n lie in it, in values; steps: its rank steps.
__device__ __forceinline__ const char* adapter_b(const AdapterArgs& e, const AdapterJob& j, int slot) {
    return static_cast<const char*>(j.b) + slot * adapter_b_slot(j.out, j.max_rank) * adapter_elem(e.type);
}
__device__ __forceinline__ uint32_t adapter_b_at(int n, int r, int steps) {
    return ((uint32_t)((n >> 4) * steps + (r >> 4)) * 64u + (uint32_t)((r & 12) << 2) + (uint32_t)(n & 15)) * 4u;
}

// sum + sum_r low[r] B[slot][n][r] over the kRanks ranks from r0 on of one row and output, r0 below the row's; low: the row's
// staged products. All of B's values are loaded before the first is used. n < j.out.
template <int kRanks>
__device__ __forceinline__ float adapter_dot(const AdapterArgs& e, const AdapterJob& j, AdapterRow row, int n, const float* low,
                                             int r0, float sum) {
    const int end = row.pad() - r0, steps = adapter_tiles16(row.pad());
    const char* b = adapter_b(e, j, row.slot());
    u32x4 w[kRanks / 4];
#pragma unroll
    for (int q = 0; q < kRanks / 4; q++) {
        const char* at = b + (size_t)adapter_b_at(n, 4 * q < end ? r0 + 4 * q : r0, steps) * adapter_elem(e.type);
        if (e.type == kAdapterF32) {
            w[q] = *reinterpret_cast<const u32x4*>(at);
        } else {
            const u32x2 v = *reinterpret_cast<const u32x2*>(at);
            w[q] = u32x4{v.x, v.y, 0u, 0u};
        }
    }
#pragma unroll
    for (int q = 0; q < kRanks / 4; q++) {
        const adapter_f32x4 l = *reinterpret_cast<const adapter_f32x4*>(low + 4 * q);
        const adapter_f32x4 f = adapter_widen4(e.type, w[q]);
#pragma unroll
        for (int i = 0; i < 4; i++) sum = 4 * q < end ? fmaf(l[i], f[i], sum) : sum;
    }
    return sum;
}

// The adapters' part of a wave's outputs in the MFMA result layout: T tiles of 16 rows from m0 on and kN tiles of 16 outputs
// from n0 on, lane (g, l16) holding rows 4 g .. 4 g + 3 of output l16 of each. All waves of the workgroup share the rows and call
// load() and add() together.
template <int T, int kN>
struct AdapterTiles {
    uint32_t key[T];  // of row m0 + 16 t + l16
    float scale[T];

    // LDS floats that add() wants
    static constexpr int kPass = 32;  // ranks staged at a time
    static constexpr int kLds = 16 * T * (kPass + 4);

    __device__ __forceinline__ void load(const AdapterArgs& e, const AdapterJob& j, int m0) {
#pragma unroll
        for (int t = 0; t < T; t++) {
            const AdapterRow r = adapter_row(e, j, m0 + 16 * t + (int)(threadIdx.x & 15));
            key[t] = r.key;
            scale[t] = r.scale;
        }
    }

    // Takes the next slot out of `left`: its rows of each tile, its key and scale; no rows if none is left.
    __device__ __forceinline__ void take(uint32_t (&left)[T], uint32_t (&rows)[T], uint32_t& k, float& s) const {
        bool found = false;
        k = 0;
        s = 0.0f;
#pragma unroll
        for (int t = 0; t < T; t++) {
            if (!found && left[t]) {
                const int l = __builtin_ctz(left[t]);
                k = (uint32_t)__builtin_amdgcn_readlane((int)key[t], l);
                s = as_float((uint32_t)__builtin_amdgcn_readlane((int)__builtin_bit_cast(uint32_t, scale[t]), l));
                found = true;
            }
        }
#pragma unroll
        for (int t = 0; t < T; t++) {
            rows[t] = found ? (uint32_t)__ballot(key[t] == k) & left[t] : 0u;
            left[t] &= ~rows[t];
        }
    }

    // out[t][c][i] += scale * (B low) for the rows that have an adapter.
    template <int kThreads>
    __device__ __forceinline__ void add(const AdapterArgs& e, const AdapterJob& j, int m0, int n0, float (&out)[T][kN][4],
                                        float* lds) const {
        constexpr uint32_t kAbsent = 0xf0000000u;  // past every resource: reads zeros
        constexpr int kRow = kPass + 4;
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
        uint32_t left[T], any = 0;
        int most = 0;  // the largest padded rank
#pragma unroll
        for (int t = 0; t < T; t++) {
            left[t] = (uint32_t)__ballot((key[t] & 0xffffu) != 0) & 0xffffu;
            any |= left[t];
            most = max(most, (int)(key[t] & 0xffffu));
        }
        if (!any) return;
        AdapterStage<16 * T, kPass, kThreads> staged;
        staged.load(e, j, m0, 0);
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) most = max(most, __shfl_xor(most, off, 64));
        most = __builtin_amdgcn_readfirstlane(most);
        uint32_t rows[2][T], k2[2];
        float s2[2];
        take(left, rows[0], k2[0], s2[0]);
        take(left, rows[1], k2[1], s2[1]);
        any = 0;
#pragma unroll
        for (int t = 0; t < T; t++) any |= left[t];
        if (any) {  // more than two slots: output by output
            float sum[T][kN][4];
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int c = 0; c < kN; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) sum[t][c][i] = 0.0f;
            for (int r0 = 0; r0 < most; r0 += kPass) {
                if (r0) {
                    adapter_barrier();
                    staged.load(e, j, m0, r0);
                }
                staged.store(e, j, m0, r0, lds);
                adapter_barrier();
#pragma unroll
                for (int t = 0; t < T; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int src = 4 * g + i;
                        const AdapterRow r{(uint32_t)__shfl((int)key[t], src, 64), 0.0f};
#pragma unroll
                        for (int c = 0; c < kN; c++)
                            if (r.pad() > r0 && n0 + 16 * c + l16 < j.out) {
                                const float* low = lds + (16 * t + src) * kRow;
                                sum[t][c][i] = most <= r0 + 16 ? adapter_dot<16>(e, j, r, n0 + 16 * c + l16, low, r0, sum[t][c][i])
                                                               : adapter_dot<32>(e, j, r, n0 + 16 * c + l16, low, r0, sum[t][c][i]);
                            }
                    }
            }
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t k = (uint32_t)__shfl((int)key[t], 4 * g + i, 64);
                    const float s = __shfl(scale[t], 4 * g + i, 64);
#pragma unroll
                    for (int c = 0; c < kN; c++)
                        if (k & 0xffffu) out[t][c][i] = fmaf(sum[t][c][i], s, out[t][c][i]);
                }
            return;
        }
        adapter_f32x4 acc[2][T][kN];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int c = 0; c < kN; c++) acc[b][t][c] = adapter_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int pad[2] = {(int)(k2[0] & 0xffffu), (int)(k2[1] & 0xffffu)};
        __amdgpu_buffer_rsrc_t br[2];
#pragma unroll
        for (int b = 0; b < 2; b++)
            br[b] = make_rsrc(adapter_b(e, j, (int)(k2[b] >> 16)),
                              (uint32_t)(adapter_tiles16(j.out) * adapter_tiles16(pad[b]) * 256 * adapter_elem(e.type)));
        for (int r0 = 0; r0 < most; r0 += kPass) {
            u32x4 raw[2][kPass / 16][kN];
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int h = 0; h < kPass / 16; h++)
#pragma unroll
                    for (int c = 0; c < kN; c++) {
                        const int n = n0 + 16 * c + l16, at = r0 + 16 * h + 4 * g;  // this lane's four ranks
                        raw[b][h][c] = adapter_load4(e.type, br[b],
                                                     at < pad[b] ? adapter_b_at(n, at, adapter_tiles16(pad[b])) *
                                                                       (uint32_t)adapter_elem(e.type)
                                                                 : kAbsent);
                    }
            if (r0) {
                adapter_barrier();
                staged.load(e, j, m0, r0);
            }
            staged.store(e, j, m0, r0, lds);
            adapter_barrier();
#pragma unroll
            for (int h = 0; h < kPass / 16; h++) {
                if (r0 + 16 * h >= most) break;
                adapter_f32x4 low[T];
#pragma unroll
                for (int t = 0; t < T; t++)
                    low[t] = *reinterpret_cast<const adapter_f32x4*>(lds + (16 * t + l16) * kRow + 16 * h + 4 * g);
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    if (r0 + 16 * h >= pad[b]) continue;
#pragma unroll
                    for (int c = 0; c < kN; c++) {
                        const adapter_f32x4 w = adapter_widen4(e.type, raw[b][h][c]);
#pragma unroll
                        for (int t = 0; t < T; t++) {
                            if (!rows[b][t]) continue;
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                acc[b][t][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(low[t][i], w[i], acc[b][t][c], 0, 0, 0);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int t = 0; t < T; t++)
#pragma unroll
                for (int c = 0; c < kN; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (rows[b][t] >> (4 * g + i) & 1) out[t][c][i] = fmaf(acc[b][t][c][i], s2[b], out[t][c][i]);
    }
};

}  // namespace ovfq
