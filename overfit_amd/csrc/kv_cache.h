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

// Walks the requests 64 at a time with `count(r)` items each (every lane of a wave calls it) until item number `item`; false past the
// last one. r: its request; item: its number within it; before: the items of the requests before r.
template <class Count>
__device__ __forceinline__ bool kv_find(int requests, int& item, int& r, int& before, Count count) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int base = 0; base < requests; base += 64) {
        const int mine = base + lane < requests ? count(base + lane) : 0;
        int upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(upto, off, 64);
            if (lane >= off) upto += v;
        }
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

}  // namespace ovfq
