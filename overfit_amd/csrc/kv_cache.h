// kv_cache.h — where a paged cache's keys and values lie, and which row belongs to which request.
//
// A block holds kKvBlock = 32 consecutive tokens of one key head, keys first, then values, in the order in which the attention
// kernels' MFMAs (16x16x32: eight contraction elements a lane) take them, so that a wave's load of an operand is 1 KiB in a row and
// nothing is transposed on the way:
//   keys    for each 16 tokens and 32 channels: lane 16 g + token holds channels 8 g .. 8 g + 7
//   values  for each 16 channels: lane 16 g + channel holds tokens 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3, which are the tokens
//           whose probabilities that lane group has after the first product: they never leave their lanes
// int8 caches hold two such pieces in a lane's 16 bytes, as quant + 128, and the tokens' 32 + 32 fp32 scales behind them.
#pragma once

#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

constexpr int kKvF16 = 1, kKvBf16 = 30, kKvI8 = 24;

__host__ __device__ constexpr int kv_plane_bytes(int type, int dp) { return dp * kKvBlock * (type == kKvI8 ? 1 : 2); }
__host__ __device__ constexpr int kv_bytes(int type, int dp) {
    return 2 * kv_plane_bytes(type, dp) + (type == kKvI8 ? 2 * kKvBlock * 4 : 0);
}

// Byte of the eight channels d8 .. d8 + 7 of token t in a block (int8: eight bytes, else sixteen).
__device__ __forceinline__ int kv_key_at(bool i8, int dp, int t, int d8) {
    const int lane = ((d8 >> 3) & 3) * 16 + (t & 15);
    if (i8) return ((((t >> 4) * (dp >> 6) + (d8 >> 6)) * 64 + lane) << 4) + ((d8 >> 5) & 1) * 8;
    return (((t >> 4) * (dp >> 5) + (d8 >> 5)) * 64 + lane) << 4;
}
// Byte of channel d of token t in a block's values.
__device__ __forceinline__ int kv_value_at(bool i8, int t, int d) {
    const int lane = ((t >> 2) & 3) * 16 + (d & 15), slot = ((t >> 4) << 2) + (t & 3);
    if (i8) return (((d >> 5) * 64 + lane) << 4) + ((d >> 4) & 1) * 8 + slot;
    return ((((d >> 4) * 64 + lane) << 4)) + slot * 2;
}
__device__ __forceinline__ char* kv_block(const KvPool& p, int page, int head, int block) {
    return p.mem + ((size_t)((int64_t)page * p.kv_heads + head) * (size_t)(p.page / kKvBlock) + block) * (size_t)kv_bytes(p.type, p.dp);
}

// Request r's rows: [first, first + n), n = 0 where its offsets do not grow or leave the rows.
struct KvRows {
    int first, n;
};
__device__ __forceinline__ KvRows kv_rows(const KvBatch& b, int r) {
    const int lo = b.row_offsets[r], hi = b.row_offsets[r + 1];
    return lo >= 0 && hi > lo && hi <= b.rows ? KvRows{lo, hi - lo} : KvRows{0, 0};
}

__device__ __forceinline__ int kv_length(const KvBatch& b, int r) { return max(b.lengths[r], 0); }

// Across a wave's lanes without LDS: the other 16 or 32 lanes' value comes from a swap of rows, neighbours' from DPP.
template <class F>
__device__ __forceinline__ int join16(int v, F f) {  // lanes l, l ^ 16
    const auto p = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    return f((int)p[0], (int)p[1]);
}
template <class F>
__device__ __forceinline__ int join32(int v, F f) {  // lanes l, l ^ 32
    const auto p = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    return f((int)p[0], (int)p[1]);
}
template <class F>
__device__ __forceinline__ int wave_join(int v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));  // row_half_mirror
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false));  // row_mirror
    return __builtin_amdgcn_readfirstlane(join32(join16(v, f), f));
}
__device__ __forceinline__ int wave_sum(int v) {
    return wave_join(v, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_max(int v) {
    return wave_join(v, [](int a, int b) { return a > b ? a : b; });
}
__device__ __forceinline__ float wave_sum(float v) {
    return as_float((uint32_t)wave_join((int)__builtin_bit_cast(uint32_t, v), [](int a, int b) {
        return (int)__builtin_bit_cast(uint32_t, as_float((uint32_t)a) + as_float((uint32_t)b));
    }));
}
// Inclusive running sum.
__device__ __forceinline__ int wave_upto(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    const int row = (int)(threadIdx.x >> 4) & 3, a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31),
              c = __builtin_amdgcn_readlane(v, 47);
    return v + (row > 0 ? a : 0) + (row > 1 ? b : 0) + (row > 2 ? c : 0);
}

// Walks the requests 64 at a time with `count(r)` items each (every lane of a wave calls it) until item number `item`; false past the
// last one. r: its request; item: its number within it; before: the items of the requests before r.
template <class Count>
__device__ __forceinline__ bool kv_find(int requests, int& item, int& r, int& before, Count count) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int base = 0; base < requests; base += 64) {
        const int mine = base + lane < requests ? count(base + lane) : 0;
        const int upto = wave_upto(mine);
        const int all = __builtin_amdgcn_readlane(upto, 63);
        if (item < before + all) {
            const int l = __ffsll((unsigned long long)__ballot(before + upto > item)) - 1;
            r = __builtin_amdgcn_readfirstlane(base + l);
            before += __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l);
            item -= before;
            return true;
        }
        before += all;
    }
    return false;
}

// The request of at most `most` rows that a row belongs to (r -1: none), every wave for itself.
struct KvRowPlace {
    int r, place;  // place: the row's token
    bool first;    // the request's first row
};
__device__ __forceinline__ KvRowPlace kv_row_place(const KvBatch& b, int row, int most) {
    const int lane = threadIdx.x & 63;
    KvRowPlace at{-1, -1, false};
    auto among = [&](int base) {  // 64 requests
        KvRows m{0, 0};
        int len = 0;
        if (base + lane < b.requests) {
            m = kv_rows(b, base + lane);
            len = kv_length(b, base + lane);
        }
        const uint64_t votes = __ballot(m.n && m.n <= most && row >= m.first && row - m.first < m.n);
        if (!votes) return false;
        const int l = __ffsll((unsigned long long)votes) - 1;
        at = KvRowPlace{__builtin_amdgcn_readfirstlane(base + l), __builtin_amdgcn_readlane(len - m.n + (row - m.first), l),
                        __builtin_amdgcn_readlane(m.first, l) == row};
        return true;
    };
    if (b.requests <= 64) {
        among(0);
        return at;
    }
    // where the row is if every request has one row; where the offsets lie around it; where offsets fall, all of them
    if (among(min(row, b.requests - 1) & ~63)) return at;
    int from = 0;
    for (int step = b.requests > 4096 ? 4096 : 64;; step = 64) {
        const int i = from + lane * step;
        const uint64_t votes = __ballot(i < b.requests && b.row_offsets[min(i, b.requests)] <= row);
        if (votes) from += (63 - __builtin_clzll(votes)) * step;
        if (step == 64) break;
    }
    if (among(from)) return at;
    for (int base = 0; base < b.requests; base += 64)
        if (among(base)) return at;
    return at;
}

}  // namespace ovfq
