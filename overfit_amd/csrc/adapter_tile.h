// adapter_tile.h — B times the rows' low-rank products in the epilogues of the projection kernels (AdapterTiles: MFMA result layout;
// AdapterOuts: a thread's outputs, the split kernels; AdapterLanes: the decode kernels), and what the launch that adds adapters to
// finished outputs shares with them (adapters.hip). Products and sums are fp32 whatever the adapters are kept in.
//
// Rows share a multiplication only where they share the slot. Tiles of few slots (a prompt's): the slots in turn, each multiplied
// over fp32 MFMA (16x16x4) with the tile's rows, and its results go to its own rows only, by selection and not by a zero factor, so
// that an infinity in one request's adapter stays out of the others' rows. Tiles of many (a decode step's): row by row, each
// output's lane with the row of B that its slot names, so that the loads are in flight together, where the walk over the slots
// waits for each group of them.
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

// Whether a tile goes row by row: its slot changes more than `few` times from row to row. key: of the tile's row l16.
__device__ __forceinline__ bool adapter_many(uint32_t key, int few) {
    const uint32_t above = (uint32_t)__builtin_amdgcn_update_dpp((int)key, (int)key, 0x111, 0xf, 0xf, false);  // row_shr:1
    return __builtin_popcount((uint32_t)__ballot(key != above) & 0xffffu) > few;
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
    // The bytes of the products from row m0 on, 0 where m0 is past the rows: loads past them read zeros.
    __device__ __forceinline__ static uint32_t held(const AdapterArgs& e, int m0) {
        const int left = e.rows - m0;
        return (uint32_t)(left < 0 ? 0 : left < kRows ? left : kRows) * (uint32_t)e.low_stride * 4u;
    }
    __device__ __forceinline__ void load(const AdapterArgs& e, const AdapterJob& j, int m0, int r0, int sh0 = 0) {
        const uint32_t bytes = held(e, m0);
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
    // load() and store() in fewer registers: a quad at a time.
    __device__ __forceinline__ static void fill(const AdapterArgs& e, const AdapterJob& j, int m0, int r0, float* lds) {
        const uint32_t bytes = held(e, m0);
#pragma unroll 1
        for (int i = 0; i < kPer; i++) {
            const int q = (int)threadIdx.x + kThreads * i;
            adapter_f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int sh0 = 0; sh0 < e.shares; sh0 += 4) {
                u32x4 v[4];
#pragma unroll
                for (int sh = 0; sh < 4; sh++)
                    v[sh] = ld4(make_rsrc(j.low + ((int64_t)(sh0 + sh) * e.rows + m0) * e.low_stride, sh0 + sh < e.shares ? bytes : 0u),
                                offset(e, i, r0));
#pragma unroll
                for (int sh = 0; sh < 4; sh++) sum += __builtin_bit_cast(adapter_f32x4, v[sh]);
            }
            if (q < kQuads) *reinterpret_cast<adapter_f32x4*>(lds + q / (kRanks / 4) * (kRanks + 4) + 4 * (q % (kRanks / 4))) = sum;
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

// One row's and output's values of B for the kRanks ranks from r0 on, and sum + sum_r low[r] B[slot][n][r] over them, r0 below the
// row's ranks; low: the row's staged products. All values are loaded before the first is used. n < j.out.
template <int kRanks>
struct AdapterDot {
    u32x4 w[kRanks / 4];

    __device__ __forceinline__ void load(const AdapterArgs& e, const AdapterJob& j, AdapterRow row, int n, int r0) {
        const int end = row.pad() - r0, steps = adapter_tiles16(row.pad());
        const char* b = adapter_b(e, j, row.slot());
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
    }
    __device__ __forceinline__ float add(const AdapterArgs& e, AdapterRow row, const float* low, int r0, float sum) const {
        const int end = row.pad() - r0;
#pragma unroll
        for (int q = 0; q < kRanks / 4; q++) {
            const adapter_f32x4 l = *reinterpret_cast<const adapter_f32x4*>(low + 4 * q);
            const adapter_f32x4 f = adapter_widen4(e.type, w[q]);
#pragma unroll
            for (int i = 0; i < 4; i++) sum = 4 * q < end ? fmaf(l[i], f[i], sum) : sum;
        }
        return sum;
    }
};
template <int kRanks>
__device__ __forceinline__ float adapter_dot(const AdapterArgs& e, const AdapterJob& j, AdapterRow row, int n, const float* low,
                                             int r0, float sum) {
    AdapterDot<kRanks> b;
    b.load(e, j, row, n, r0);
    return b.add(e, row, low, r0, sum);
}

// The same in eight registers: 16 ranks of the 16-bit types, 8 of fp32.
struct AdapterOct {
    u32x4 w[2];

    __device__ __forceinline__ static int ranks(const AdapterArgs& e) { return e.type == kAdapterF32 ? 8 : 16; }
    __device__ __forceinline__ void load(const AdapterArgs& e, const AdapterJob& j, AdapterRow row, int n, int r0) {
        const int end = row.pad() - r0, steps = adapter_tiles16(row.pad());
        const char* b = adapter_b(e, j, row.slot());
        auto at = [&](int q) {
            return b + (size_t)adapter_b_at(n, 4 * q < end ? r0 + 4 * q : r0, steps) * adapter_elem(e.type);
        };
        if (e.type == kAdapterF32) {
#pragma unroll
            for (int q = 0; q < 2; q++) w[q] = *reinterpret_cast<const u32x4*>(at(q));
        } else {
            u32x2 v[4];
#pragma unroll
            for (int q = 0; q < 4; q++) v[q] = *reinterpret_cast<const u32x2*>(at(q));
#pragma unroll
            for (int q = 0; q < 2; q++) w[q] = u32x4{v[2 * q].x, v[2 * q].y, v[2 * q + 1].x, v[2 * q + 1].y};
        }
    }
    __device__ __forceinline__ float add(const AdapterArgs& e, AdapterRow row, const float* low, int r0, float sum) const {
        const int end = row.pad() - r0;
        auto quad = [&](int q, u32x4 v) {
            const adapter_f32x4 l = *reinterpret_cast<const adapter_f32x4*>(low + 4 * q);
            const adapter_f32x4 f = adapter_widen4(e.type, v);
#pragma unroll
            for (int i = 0; i < 4; i++) sum = 4 * q < end ? fmaf(l[i], f[i], sum) : sum;
        };
        if (e.type == kAdapterF32) {
#pragma unroll
            for (int q = 0; q < 2; q++) quad(q, w[q]);
        } else {
#pragma unroll
            for (int q = 0; q < 2; q++) {
                quad(2 * q, u32x4{w[q].x, w[q].y, 0u, 0u});
                quad(2 * q + 1, u32x4{w[q].z, w[q].w, 0u, 0u});
            }
        }
        return sum;
    }
};

// The adapters' part of a wave's outputs in the MFMA result layout: T tiles of 16 rows from m0 on and kN tiles of 16 outputs
// from n0 on, lane (g, l16) holding rows 4 g .. 4 g + 3 of output l16 of each. All waves of the workgroup share the rows and call
// load() and add() together. kPass: ranks staged at a time. kAhead: slots whose B values are loaded together. kTiles: row tiles
// that go row by row at a time; 0: none do (that takes more registers than the tiled kernels have), and those that would are left
// to the launch behind where there is one (by_row).
template <int T, int kN, int kPass = 32, int kAhead = 1, int kTiles = 0>
struct AdapterTiles {
    uint32_t key[T];  // of row m0 + 16 t + l16
    float scale[T];

    // LDS floats that add() wants
    static constexpr int kRow = kPass + 4, kScale = 16 * T * kRow, kLds = kScale + 16 * T;

    __device__ __forceinline__ void load(const AdapterArgs& e, const AdapterJob& j, int m0) {
#pragma unroll
        for (int t = 0; t < T; t++) {
            const AdapterRow r = adapter_row(e, j, m0 + 16 * t + (int)(threadIdx.x & 15));
            key[t] = r.key;
            scale[t] = r.scale;
            if (e.by_row && adapter_many(key[t], e.by_row)) key[t] = 0;  // the launch behind has this tile
        }
    }

    // Takes the next slot out of `left`: its rows of each tile, and its key; no rows and 0 if none is left.
    __device__ __forceinline__ uint32_t take(uint32_t (&left)[T], uint32_t (&rows)[T]) const {
        uint32_t k = 0;
#pragma unroll
        for (int t = 0; t < T; t++)
            if (!k && left[t]) k = (uint32_t)__builtin_amdgcn_readlane((int)key[t], __builtin_ctz(left[t]));
#pragma unroll
        for (int t = 0; t < T; t++) {
            rows[t] = (uint32_t)__ballot(key[t] == k) & left[t];
            left[t] &= ~rows[t];
        }
        return k;
    }

    // The lane's B values of ranks r0 .. r0 + kPass and the outputs from n0 on; zeros past the slot's ranks.
    __device__ __forceinline__ static void load_b(const AdapterArgs& e, const AdapterJob& j, uint32_t k, int n0, int r0,
                                                  u32x4 (&raw)[kPass / 16][kN]) {
        constexpr uint32_t kAbsent = 0xf0000000u;  // past every resource: reads zeros
        const int lane = threadIdx.x & 63, pad = (int)(k & 0xffffu), steps = adapter_tiles16(pad);
        const __amdgpu_buffer_rsrc_t br = make_rsrc(adapter_b(e, j, (int)(k >> 16)),
                                                    (uint32_t)(adapter_tiles16(j.out) * steps * 256 * adapter_elem(e.type)));
#pragma unroll
        for (int h = 0; h < kPass / 16; h++)
#pragma unroll
            for (int c = 0; c < kN; c++) {
                const int at = r0 + 16 * h + 4 * (lane >> 4);  // this lane's four ranks
                raw[h][c] = adapter_load4(e.type, br,
                                          at < pad ? adapter_b_at(n0 + 16 * c + (lane & 15), at, steps) * (uint32_t)adapter_elem(e.type)
                                                   : kAbsent);
            }
    }

    // sum += B low of the ranks from r0 on for the tiles in `by_row`.
    __device__ __forceinline__ void row_by_row(const AdapterArgs& e, const AdapterJob& j, int n0, int r0, int most, const float* lds,
                                               const bool (&by_row)[T], adapter_f32x4 (&sum)[T][kN]) const {
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
        const int step = AdapterOct::ranks(e), ranks = most - r0 < kPass ? most - r0 : kPass;
#pragma unroll
        for (int t0 = 0; t0 < T; t0 += kTiles) {
            bool any = false;
#pragma unroll
            for (int t = t0; t < T && t < t0 + kTiles; t++) any = any || by_row[t];
            if (!any) continue;
#pragma unroll
            for (int c = 0; c < kN; c++) {
                const int n = n0 + 16 * c + l16;
                AdapterRow row[kTiles][4];
#pragma unroll
                for (int t = 0; t < kTiles && t0 + t < T; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        row[t][i] = AdapterRow{(uint32_t)__shfl((int)key[t0 + t], 4 * g + i, 64), 0.0f};
                        if (!by_row[t0 + t] || n >= j.out) row[t][i].key = 0;
                    }
#pragma unroll 1
                for (int h = 0; h < ranks; h += step) {
                    AdapterOct b[kTiles][4];
#pragma unroll
                    for (int t = 0; t < kTiles && t0 + t < T; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (row[t][i].pad() > r0 + h) b[t][i].load(e, j, row[t][i], n, r0 + h);
#pragma unroll
                    for (int t = 0; t < kTiles && t0 + t < T; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (row[t][i].pad() > r0 + h)
                                sum[t0 + t][c][i] = b[t][i].add(e, row[t][i], lds + (16 * (t0 + t) + 4 * g + i) * kRow + h, r0 + h,
                                                                sum[t0 + t][c][i]);
                }
            }
        }
    }

    // out[t][c][i] += scale * (B low) for the rows that have an adapter. The products of all rows with a slot's B go on from the
    // sums, and the slot's own rows keep them.
    template <int kThreads>
    __device__ __forceinline__ void add(const AdapterArgs& e, const AdapterJob& j, int m0, int n0, float (&out)[T][kN][4],
                                        float* lds) const {
        using Stage = AdapterStage<16 * T, kPass, kThreads>;
        const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
        Stage staged;
        staged.load(e, j, m0, 0);
        uint32_t left[T], any = 0;
        bool by_row[T];
        int most = 0;  // the largest padded rank
#pragma unroll
        for (int t = 0; t < T; t++) {
            left[t] = (uint32_t)__ballot((key[t] & 0xffffu) != 0) & 0xffffu;
            any |= left[t];
            most = max(most, (int)(key[t] & 0xffffu));
            by_row[t] = false;
            if constexpr (kTiles > 0) by_row[t] = j.slots > kAdapterFew && adapter_many(key[t], kAdapterFew);
            if (by_row[t]) left[t] = 0;
        }
        if (!any) return;
        uint32_t k[kAhead], rows[kAhead][T];
        u32x4 raw[kAhead][kPass / 16][kN];
        auto next = [&](int r0) {  // the next slots' rows, keys and B values
#pragma unroll
            for (int b = 0; b < kAhead; b++) {
                k[b] = take(left, rows[b]);
                if (k[b]) load_b(e, j, k[b], n0, r0, raw[b]);
            }
        };
        next(0);
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) most = max(most, __shfl_xor(most, off, 64));
        most = __builtin_amdgcn_readfirstlane(most);
        staged.store(e, j, m0, 0, lds);
        if (threadIdx.x < 16) {
#pragma unroll
            for (int t = 0; t < T; t++) lds[kScale + 16 * t + l16] = scale[t];
        }
        adapter_f32x4 sum[T][kN];
#pragma unroll
        for (int t = 0; t < T; t++)
#pragma unroll
            for (int c = 0; c < kN; c++) sum[t][c] = adapter_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (int r0 = 0;;) {
            adapter_barrier();
#pragma unroll 1
            while (k[0]) {
#pragma unroll
                for (int b = 0; b < kAhead; b++) {
                    const int ranks = (int)(k[b] & 0xffffu) - r0;
                    if (ranks <= 0) break;  // no slot
                    adapter_f32x4 w[kPass / 16][kN];
#pragma unroll
                    for (int h = 0; h < kPass / 16; h++)
#pragma unroll
                        for (int c = 0; c < kN; c++) w[h][c] = adapter_widen4(e.type, raw[b][h][c]);
#pragma unroll
                    for (int t = 0; t < T; t++) {
                        if (!rows[b][t]) continue;
                        adapter_f32x4 acc[kN];
#pragma unroll
                        for (int c = 0; c < kN; c++) acc[c] = sum[t][c];
#pragma unroll
                        for (int h = 0; h < kPass / 16; h++) {
                            if (16 * h >= ranks) continue;
                            const adapter_f32x4 low =
                                *reinterpret_cast<const adapter_f32x4*>(lds + (16 * t + l16) * kRow + 16 * h + 4 * g);
#pragma unroll
                            for (int c = 0; c < kN; c++)
#pragma unroll
                                for (int i = 0; i < 4; i++)
                                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(low[i], w[h][c][i], acc[c], 0, 0, 0);
                        }
#pragma unroll
                        for (int c = 0; c < kN; c++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (rows[b][t] >> (4 * g + i) & 1) sum[t][c][i] = acc[c][i];
                    }
                }
                next(r0);
            }
            if constexpr (kTiles > 0) row_by_row(e, j, n0, r0, most, lds, by_row, sum);
            r0 += kPass;
            if (r0 >= most) break;
#pragma unroll
            for (int t = 0; t < T; t++) left[t] = by_row[t] ? 0u : (uint32_t)__ballot((int)(key[t] & 0xffffu) > r0) & 0xffffu;
            next(r0);
            adapter_barrier();
            Stage::fill(e, j, m0, r0, lds);
        }
#pragma unroll
        for (int t = 0; t < T; t++) {
            const adapter_f32x4 s = *reinterpret_cast<const adapter_f32x4*>(lds + kScale + 16 * t + 4 * g);
            const uint32_t has = (uint32_t)__ballot((key[t] & 0xffffu) != 0);
#pragma unroll
            for (int c = 0; c < kN; c++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (has >> (4 * g + i) & 1) out[t][c][i] = fmaf(sum[t][c][i], s[i], out[t][c][i]);
        }
    }
};

// add() for out[T][4] and one output tile, kBy row tiles at a time (the registers that T at once would take).
template <int T, int kBy, int kPass, int kThreads, int kAhead = 1>
__device__ __forceinline__ void adapter_add(const AdapterArgs& e, const AdapterJob& j, int m0, int n0, float (&out)[T][4], float* lds) {
    static_assert(T % kBy == 0, "whole groups of tiles");
#pragma unroll
    for (int t0 = 0; t0 < T; t0 += kBy) {
        AdapterTiles<kBy, 1, kPass, kAhead> tiles;
        tiles.load(e, j, m0 + 16 * t0);
        float v[kBy][1][4];
#pragma unroll
        for (int t = 0; t < kBy; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[t][0][i] = out[t0 + t][i];
        if (t0) adapter_barrier();  // the last tiles' products have been read
        tiles.template add<kThreads>(e, j, m0 + 16 * t0, n0, v, lds);
#pragma unroll
        for (int t = 0; t < kBy; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) out[t0 + t][i] = v[t][0][i];
    }
}

// The adapters' part of a workgroup's 16 T rows x 16 outputs, its 64 W threads each taking the outputs threadIdx.x + 64 W i: output
// (idx >> 4) & 15 of row (idx >> 8) * 16 + (idx & 15). Every output loads the row of B that its slot names, so that all loads are in
// flight at once, however many slots the rows have. kLowPass: ranks staged at a time.
template <int T, int W, int kLowPass>
struct AdapterOuts {
    static constexpr int kPer = (256 * T + 64 * W - 1) / (64 * W);  // (past the rows: no row has a key there)
    static constexpr int kLds = 16 * T * (kLowPass + 4);  // floats of `staged`
    static constexpr int kAtOnce = kPer == 1 ? kLowPass : 32;  // ranks of B in registers at once
    AdapterTiles<T, 1> rows;
    AdapterStage<16 * T, kLowPass, 64 * W> stage;

    __device__ __forceinline__ void load(const AdapterArgs& e, const AdapterJob& j, int m0) {
        rows.load(e, j, m0);
        stage.load(e, j, m0, 0);
    }

    // kRanks of every output of the thread from r0 on, all outputs' values of B loaded together; first: the products are staged too.
    template <int kRanks>
    __device__ __forceinline__ void together(const AdapterArgs& e, const AdapterJob& j, const AdapterRow (&row)[kPer], int o0, int r0,
                                             bool first, float* staged, float (&sum)[kPer], int m0) {
        AdapterDot<kRanks> b[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (row[i].pad() > r0) b[i].load(e, j, row[i], o0 + ((((int)threadIdx.x + 64 * W * i) >> 4) & 15), r0);
        if (first) {
            stage.store(e, j, m0, r0, staged);
            adapter_barrier();
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int idx = (int)threadIdx.x + 64 * W * i;
            const float* low = staged + ((idx >> 8) * 16 + (idx & 15)) * (kLowPass + 4) + r0 % kLowPass;
            if (row[i].pad() > r0) sum[i] = b[i].add(e, row[i], low, r0, sum[i]);
        }
    }

    // Leaves the thread's parts in out[idx] and returns which of its outputs have one. All waves; `staged` is free again after.
    __device__ __forceinline__ uint32_t part(const AdapterArgs& e, const AdapterJob& j, int m0, int o0, float* staged, float* out) {
        AdapterRow row[kPer];
        float sum[kPer];
        int most = 0;  // the largest padded rank of the workgroup's rows, the same for every wave
#pragma unroll
        for (int t = 0; t < T; t++) most = max(most, (int)(rows.key[t] & 0xffffu));
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) most = max(most, __shfl_xor(most, off, 64));
        most = __builtin_amdgcn_readfirstlane(most);
#pragma unroll
        for (int i = 0; i < kPer; i++) {  // (a wave's outputs are of one row tile)
            const int idx = (int)threadIdx.x + 64 * W * i;
            row[i] = AdapterRow{0, 0.0f};
#pragma unroll
            for (int t = 0; t < T; t++)
                if ((wave_id() + W * i) >> 2 == t) row[i] = AdapterRow{rows.key[t], rows.scale[t]};
            if (o0 + ((idx >> 4) & 15) >= j.out) row[i].key = 0;
            sum[i] = 0.0f;
        }
        for (int r0 = 0; r0 < most; r0 += kLowPass) {
            if (r0) {
                adapter_barrier();
                stage.load(e, j, m0, r0);
            }
            if constexpr (T <= 2) {
                // B's first values are under way while the products are staged (down 14336 -> 4096, 7 rows of rank 64: the kernel
                // 21.9 -> 21.1 us; with three and four row tiles the registers spill, 64 rows of 4096 -> 4096 19.8 -> 21.9)
                const int left = most - r0;  // the same for every wave
                if (left <= 16)
                    together<16>(e, j, row, o0, r0, true, staged, sum, m0);
                else if (left <= 32 || kAtOnce == 32)
                    for (int h = 0; h < kLowPass && h < left; h += 32) together<32>(e, j, row, o0, r0 + h, !h, staged, sum, m0);
                else
                    together<kAtOnce>(e, j, row, o0, r0, true, staged, sum, m0);
                continue;
            }
            stage.store(e, j, m0, r0, staged);
            adapter_barrier();
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                const int idx = (int)threadIdx.x + 64 * W * i, n = o0 + ((idx >> 4) & 15);
                const float* low = staged + ((idx >> 8) * 16 + (idx & 15)) * (kLowPass + 4);
#pragma unroll
                for (int h = 0; h < kLowPass; h += 32) {
                    if (r0 + h >= most) break;  // the same for every wave
                    if (row[i].pad() > r0 + h)
                        sum[i] = most <= r0 + h + 16 ? adapter_dot<16>(e, j, row[i], n, low + h, r0 + h, sum[i])
                                                     : adapter_dot<32>(e, j, row[i], n, low + h, r0 + h, sum[i]);
                }
            }
        }
        if (most) adapter_barrier();
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            if (!row[i].pad()) continue;
            out[(int)threadIdx.x + 64 * W * i] = sum[i] * row[i].scale;
            mine |= 1u << i;
        }
        return mine;
    }
};

// The adapters' part of a decode kernel's outputs: output oi of a wave's item (weight row n, activation row m) has the L lanes
// from L oi on, each with every L-th quad of the ranks. The rows' adapters are loaded at the start, a lane's first P quads of B
// beside the item's weights; the launch's low-rank products wait in LDS, [job][row][low_stride]. In launches of several weights the
// choice of key and scale by the job keeps the whole of it in private memory (176 bytes a lane): q/k/v of 4096 Q4_K, one row, rank 16
// 19.5 us, 4.4 without adapters; the output projection alone, whose kernel has none there, 9.8 and 3.9.
template <int L, int P, int kThreads>
struct AdapterLanes {
    uint32_t key[kMaxJobs];  // of the lane's activation row
    float scale[kMaxJobs];
    u32x4 part[8];  // a quad of the products, its shares

    struct Item {
        u32x4 b[P];
    };

    __device__ __forceinline__ void load_products(const AdapterArgs& e, int f) {
        const int quads = e.rows * e.low_stride / 4;  // of a job and share; the jobs' planes are one behind the other
        int j = 0;
#pragma unroll
        for (int i = 1; i < kMaxJobs; i++) j += f >= i * quads;
        const __amdgpu_buffer_rsrc_t r = make_rsrc(e.job[0].low, (uint32_t)(e.jobs * e.shares * quads) * 16u);
#pragma unroll
        for (int sh = 0; sh < 8; sh++)
            part[sh] = ld4(r, sh < e.shares && f < e.jobs * quads ? (uint32_t)((j * (e.shares - 1) + sh) * quads + f) * 16u : 0xf0000000u);
    }
    // m: the lane's activation row
    __device__ __forceinline__ void load(const AdapterArgs& e, int m) {
#pragma unroll
        for (int j = 0; j < kMaxJobs; j++) {
            const bool any = j < e.jobs && e.job[j].slots;
            const u32x2 v = ld2(make_rsrc(any ? (const void*)e.job[j].row : (const void*)e.x, any ? (uint32_t)e.rows * 8u : 0u),
                                (uint32_t)m * 8u);
            const uint32_t s = v.y;
            key[j] = v.x;
            scale[j] = as_float(s);
        }
        load_products(e, (int)threadIdx.x);
    }
    // The products into LDS; the workgroup's barrier comes after.
    __device__ __forceinline__ void stage(const AdapterArgs& e, float* low) {
        const int quads = e.jobs * e.rows * e.low_stride / 4;
        for (int f = (int)threadIdx.x;;) {
            adapter_f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int sh = 0; sh < 8; sh++) sum += __builtin_bit_cast(adapter_f32x4, part[sh]);
            if (f < quads) *reinterpret_cast<adapter_f32x4*>(low + 4 * f) = sum;
            f += kThreads;
            if (f - (int)threadIdx.x >= quads) break;  // the same for every thread
            load_products(e, f);
        }
    }

    __device__ __forceinline__ uint32_t key_of(int job) const {
        uint32_t k = key[0];
#pragma unroll
        for (int i = 1; i < kMaxJobs; i++) k = job == i ? key[i] : k;
        return k;
    }
    // Where the lane's quad q of output n lies in the B of slot `k`; a quad that is not there reads some of x, unused.
    __device__ __forceinline__ static u32x4 quad(const AdapterArgs& e, const AdapterJob& j, uint32_t k, int n, int q, bool want) {
        const int pad = (int)(k & 0xffffu);
        const bool there = want && 4 * q < pad;
        const char* at = there ? adapter_b(e, j, (int)(k >> 16)) + (size_t)adapter_b_at(n, 4 * q, adapter_tiles16(pad)) * adapter_elem(e.type)
                               : reinterpret_cast<const char*>(e.x);
        if (e.type == kAdapterF32) return *reinterpret_cast<const u32x4*>(at);
        const u32x2 v = *reinterpret_cast<const u32x2*>(at);
        return u32x4{v.x, v.y, 0u, 0u};
    }
    // Issues the loads of the lane's output n of weight `job`; always as many, so that the waits before them count on.
    __device__ __forceinline__ void fetch(const AdapterArgs& e, int job, int n, bool want, Item& it) const {
        const AdapterJob j = adapter_job(e, job);
        const uint32_t k = key_of(job);
        const int sub = (int)(threadIdx.x % L);
#pragma unroll
        for (int p = 0; p < P; p++) it.b[p] = quad(e, j, k, n, sub + L * p, want && n < j.out);
    }
    // y += scale * (B low) for output `lane` of the item; n, m: of the output that the lane works for.
    __device__ __forceinline__ void add(const AdapterArgs& e, int job, int n, int m, const Item& it, const float* low, float& y) const {
        const AdapterJob j = adapter_job(e, job);
        const uint32_t k = key_of(job);
        const int pad = (int)(k & 0xffffu), sub = (int)(threadIdx.x % L);
        const bool live = pad && m < e.rows && n < j.out;
        const float* mine = low + (size_t)(job * e.rows + (live ? m : 0)) * e.low_stride;
        float sum = 0.0f;
        auto more = [&](int q, u32x4 raw) {
            if (!live || 4 * q >= pad) return;
            const adapter_f32x4 l = *reinterpret_cast<const adapter_f32x4*>(mine + 4 * q);
            const adapter_f32x4 w = adapter_widen4(e.type, raw);
#pragma unroll
            for (int i = 0; i < 4; i++) sum = fmaf(l[i], w[i], sum);
        };
#pragma unroll
        for (int p = 0; p < P; p++) more(sub + L * p, it.b[p]);
        for (int q0 = L * P; q0 < adapter_tiles16(j.max_rank) * 4; q0 += 4 * L) {
            u32x4 raw[4];
#pragma unroll
            for (int p = 0; p < 4; p++) raw[p] = quad(e, j, k, n, q0 + sub + L * p, live);
#pragma unroll
            for (int p = 0; p < 4; p++) more(q0 + sub + L * p, raw[p]);
        }
#pragma unroll
        for (int off = L / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        float s = scale[0];
#pragma unroll
        for (int i = 1; i < kMaxJobs; i++) s = job == i ? scale[i] : s;
        const int lane = (int)(threadIdx.x & 63), src = lane * L & 63;
        const float delta = __shfl(sum * s, src, 64);
        const bool has = __shfl((int)live, src, 64) != 0;
        if (has) y += delta;
    }
};

// The LDS that AdapterLanes' products take, and whether it is left beside `lds` bytes of the kernel's own.
inline size_t adapter_lanes_lds(const AdapterArgs& e) { return (size_t)e.jobs * e.rows * e.low_stride * 4; }
inline bool adapter_lanes_fit(const AdapterArgs& e, size_t lds) { return e.shares <= 8 && lds + adapter_lanes_lds(e) <= 65536; }

}  // namespace ovfq
