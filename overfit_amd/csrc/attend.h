// attend.h — what the attention kernels over a paged cache share: their arithmetic on one block of 32 tokens, and the way the work
// is cut.
//
//   out = softmax(scale q . k) v   over the tokens j with  position - window < j <= position  (window 0: all up to the position)
//
// A kernel's columns are (row, query head) pairs of one request and key head, row by row: column c is row c / group, head c % group.
// Products are MFMA 16x16x32 with the cache's operands as the first factor, so that a lane's results belong to one column (lane % 16)
// and to the tokens whose values the same lane group loads for the second product: probabilities never change lanes.
//
// Rounding. q and p are fp32 and enter the products in parts: two fp16 ones beside fp16 and int8 operands (22 bits, for numbers down to
// 2^-14; what lies below is held to 2^-25 whatever its size), three bf16 ones beside bf16 operands (24 bits). q is scaled by a power of
// two, its row's largest channel to between 1 and 2, so a channel is off by 2^-23 of that one at most. p is 2^kTop at the largest score
// that its column has met when it last moved its reference, which it does when a score passes that by 2^kRoom: beside fp16 values
// 2^10, so that fp16 has 2^24 below the largest p and no overflow above; beside bf16 values 2^-16, so that sums over 2^12 of the largest
// values still fit fp32. Sums and references are fp32; outputs are divided by their sum before they are joined, and are never larger than
// the values.
// int8 operands are widened to fp16, which is exact. A token's key scale multiplies its scores, its value scale its p (2^2 at the
// reference, so that the product fits fp32); what enters the second product is p scale / e, with a power of two e kept for the column
// that puts the largest p scale so far between 2^10 and 2^15. Both move with the column's reference, so a large scale of little weight
// takes nothing from the others. (Against the largest scale seen, whatever its weight, a token of 2^36 times the others' scales and no
// weight made zeros of the rows that saw it. What the largest product costs: a prompt of 4096 rows 312 -> 323 us, 60 drafted rows 84.0 ->
// 84.7. A bound of it, checked with the reference, spilled registers: 419 and 503.)
//
// Masks: a hidden token's score is -inf whatever its key holds. A hidden token's value meets a probability of zero, which would still
// make NaN of what is not finite, so blocks with a mask look at their values first: what is not finite is noted for the columns that see
// it (their outputs become NaN in the end) and taken out of the operand. (Adding such tokens one by one in a path of its own doubled the
// accumulators' registers: the prompt kernel's 256 were not enough, and a spilled register's reload waits for the next block's DMA as
// well. 4100 rows of three prompts 243 us that way.)
#pragma once

#include "kv_cache.h"

namespace ovfq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ uint32_t bits_of(float v) { return __builtin_bit_cast(uint32_t, v); }  // (straight from a vector it reads element 0)

// Over the four lanes of a column: l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float column_max(float v) {
    auto f = [](int a, int b) { return (int)__builtin_bit_cast(uint32_t, fmaxf(as_float((uint32_t)a), as_float((uint32_t)b))); };
    return as_float((uint32_t)join32(join16((int)__builtin_bit_cast(uint32_t, v), f), f));
}
__device__ __forceinline__ uint32_t column_max(uint32_t v) {
    auto f = [](int a, int b) { return (int)max((uint32_t)a, (uint32_t)b); };
    return (uint32_t)join32(join16((int)v, f), f);
}
__device__ __forceinline__ float column_sum(float v) {
    auto f = [](int a, int b) { return (int)__builtin_bit_cast(uint32_t, as_float((uint32_t)a) + as_float((uint32_t)b)); };
    return as_float((uint32_t)join32(join16((int)__builtin_bit_cast(uint32_t, v), f), f));
}

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRoom = 4.0f;  // log2 of how far p may grow past a new reference before the next

template <int kType>
struct KvMath {
    static constexpr int kParts = kType == kKvBf16 ? 3 : 2;
    static constexpr float kTop = kType == kKvF16 ? 10.0f : kType == kKvBf16 ? -16.0f : 2.0f;  // log2 of p at a new reference
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        if constexpr (kType == kKvBf16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    }
    // Eight fp32 values as kParts operands that add up to them.
    static __device__ __forceinline__ void split(const float (&x)[8], u32x4 (&part)[kParts]) {
        float minus = -1.0f;
        asm("" : "+v"(minus));  // (a constant would make a conversion and a subtraction of the v_fma_mix below)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f32x2 v = {x[2 * i], x[2 * i + 1]};
#pragma unroll
            for (int p = 0; p < kParts; p++) {
                if constexpr (kType == kKvBf16) {
                    const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b16x2));
                    part[p][i] = w;
                    if (p + 1 < kParts) v = f32x2{v.x - as_float(w << 16), v.y - as_float(w & 0xffff0000u)};
                } else {
                    const h16x2 h = __builtin_convertvector(v, h16x2);
                    part[p][i] = __builtin_bit_cast(uint32_t, h);
                    if (p + 1 < kParts) v = f32x2{fmaf((float)h.x, minus, v.x), fmaf((float)h.y, minus, v.y)};
                }
            }
        }
    }
};

// Eight int8 quants (as + 128) to fp16: byte b under the exponent of 1024 is 1024 + b.
__device__ __forceinline__ u32x4 widened(uint32_t lo, uint32_t hi) {
    const h16x2 zero = {(_Float16)1152.0f, (_Float16)1152.0f};
    const uint32_t w[4] = {__builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u),
                           __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)};
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h16x2, w[i]) - zero);
    return r;
}

// Bits 15 and 31 of each word: which of an fp16 or bf16 operand's eight values are not finite.
template <int kType>
__device__ __forceinline__ u32x4 not_finite(u32x4 v) {
    constexpr uint32_t kExp = kType == kKvBf16 ? 0x7f807f80u : 0x7c007c00u, kOne = kType == kKvBf16 ? 0x00800080u : 0x04000400u;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = ((v[i] & kExp) + kOne) & 0x80008000u;
    return r;
}
template <int kType>
__device__ __forceinline__ bool any_not_finite(u32x4 v) {
    const u32x4 b = not_finite<kType>(v);
    return (b.x | b.y | b.z | b.w) != 0;
}
// The operand with zeros in their places.
template <int kType>
__device__ __forceinline__ u32x4 finite_part(u32x4 v) {
    const u32x4 b = not_finite<kType>(v);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] &= ~((b[i] >> 15) * 0xffffu);
    return v;
}

// kCols 16-column tiles of queries against a request's blocks, one wave.
template <int kType, int kDp, int kCols>
struct Attention {
    using M = KvMath<kType>;
    static constexpr int kChunks = kDp / 32, kTiles = kDp / 16;
    u32x4 q[kCols][M::kParts][kChunks];
    float qs[kCols];           // q's power of two
    int lim[kCols], low[kCols];  // the column's last token, and its first
    f32x4 o[kCols][kTiles];
    float ref[kCols], l[kCols];  // l: of this lane's tokens
    float ev[kCols];             // int8: the power of two that p times the values' scales are divided by, so o as well
    float fall[kCols];           // int8: what a new reference has made of earlier probabilities, 1 without one
    uint32_t bad[kCols][2];      // bit 4 d + i: the column sees a value that is not finite in o[][d][i]'s channel (of masked blocks)

    // A query row's channels of this lane, zeros if the column is not used.
    using Row = float[kChunks][8];
    static __device__ __forceinline__ void fetch(Row& v, const float* x, bool used, int dim) {
        const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            const int d = c * 32 + g * 8, in = d < dim ? d : 0;
            f32x4u a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (used) {
                a = *(const f32x4u*)(x + in);
                b = *(const f32x4u*)(x + in + 4);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) v[c][i] = i < 4 ? a[i & 3] : b[i & 3];
        }
    }
    // Column t of the wave, if `used`, sees the tokens [first, last].
    __device__ __forceinline__ void column(int t, bool used, int first, int last) {
        lim[t] = used ? last : -1;
        low[t] = first;
        ref[t] = -kInf;
        l[t] = 0.0f;
        ev[t] = as_float(1u << 23);
        bad[t][0] = bad[t][1] = 0;
#pragma unroll
        for (int d = 0; d < kTiles; d++) o[t][d] = f32x4{0, 0, 0, 0};
    }
    // Its query row; zeros for a column that is not used.
    __device__ __forceinline__ void query(int t, Row& v, bool used, int dim, float scale) {
        const int g = (threadIdx.x >> 4) & 3;
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[c][i] = used && c * 32 + g * 8 < dim ? v[c][i] * scale : 0.0f;
                top = fmaxf(top, fabsf(v[c][i]));
            }
        top = column_max(top);
        const int e = min(max((int)(__builtin_bit_cast(uint32_t, top) >> 23), 1), 253);
        const float down = as_float((uint32_t)(254 - e) << 23);
        qs[t] = as_float((uint32_t)e << 23);
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            float w[8];
            u32x4 part[M::kParts];
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = v[c][i] * down;
            M::split(w, part);
#pragma unroll
            for (int p = 0; p < M::kParts; p++) q[t][p][c] = part[p];
        }
    }

    // Scores of a block; key(tile, chunk): the operand of its 16 tokens and 32 channels.
    template <class Key>
    __device__ __forceinline__ void scores(f32x4 (&s)[kCols][2], Key key) {
#pragma unroll
        for (int t = 0; t < kCols; t++) s[t][0] = s[t][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kChunks; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const u32x4 a = key(h, c);
#pragma unroll
                for (int p = 0; p < M::kParts; p++)
#pragma unroll
                    for (int t = 0; t < kCols; t++) s[t][h] = M::mfma(a, q[t][p][c], s[t][h]);
            }
    }

    // Whether column t sees token j.
    __device__ __forceinline__ bool sees(int t, int j) const { return (int)(j <= lim[t]) & (int)(j >= low[t]); }

    // A block's scores before their powers: int8's key scales, masks, and the columns' references. first: the block's first token; ks:
    // int8's scales of this lane's keys.
    __device__ __forceinline__ void settle(f32x4 (&s)[kCols][2], bool masked, int first, const f32x4 (&ks)[2]) {
        const int mine = first + ((threadIdx.x >> 4) & 3) * 4;
        if constexpr (kType == kKvI8) {
#pragma unroll
            for (int t = 0; t < kCols; t++) {
                fall[t] = 1.0f;
#pragma unroll
                for (int h = 0; h < 2; h++) s[t][h] *= ks[h];
            }
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < kCols; t++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[t][h][i] = sees(t, mine + 16 * h + i) ? s[t][h][i] : -kInf;
        }
        bool move = false;
        float top[kCols];
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            top[t] = s[t][0][0];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (h + i) top[t] = fmaxf(top[t], s[t][h][i]);
            top[t] *= qs[t];
            move = move | (top[t] > ref[t] + M::kTop + kRoom);
        }
        if (__ballot(move)) {
#pragma unroll
            for (int t = 0; t < kCols; t++) {
                const float m = column_max(top[t]);
                float f = 1.0f;
                if (m > ref[t] + M::kTop + kRoom) {
                    f = __builtin_amdgcn_exp2f(ref[t] - (m - M::kTop));
                    ref[t] = m - M::kTop;
                    l[t] *= f;
                }
                if constexpr (kType == kKvI8) {
                    fall[t] = f;
                } else {
#pragma unroll
                    for (int d = 0; d < kTiles; d++) o[t][d] *= f;
                }
            }
        }
    }

    // Settled scores into probabilities (int8: times their values' scales vs), split for the second product.
    __device__ __forceinline__ void probabilities(const f32x4 (&s)[kCols][2], u32x4 (&p)[kCols][M::kParts], bool masked, int first,
                                                  const f32x4 (&vs)[2]) {
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            const float r = ref[t] == -kInf ? 0.0f : ref[t];
            float x[8];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = __builtin_amdgcn_exp2f(fmaf(s[t][h][i], qs[t], -r));
                    l[t] += v;
                    x[4 * h + i] = kType == kKvI8 ? v * vs[h][i] : v;
                }
            if constexpr (kType == kKvI8) {
                if (masked) {  // (a hidden token's scale may be anything, and its probability is 0)
                    const int mine = first + ((threadIdx.x >> 4) & 3) * 4;
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = sees(t, mine + (i >> 2) * 16 + (i & 3)) ? x[i] : 0.0f;
                }
                float top = x[0];
#pragma unroll
                for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
                if (__ballot(top > ev[t] * 16384.0f || fall[t] != 1.0f)) {
                    top = column_max(top);
                    if (top > ev[t] * 16384.0f || fall[t] != 1.0f) {
                        const float was = ev[t] * fall[t];  // what o's unit is worth now
                        const int e = min(max(max((int)(bits_of(was) >> 23), (int)(bits_of(top) >> 23) - 10), 1), 253);
                        const float f = was * as_float((uint32_t)(254 - e) << 23);
                        ev[t] = as_float((uint32_t)e << 23);
#pragma unroll
                        for (int d = 0; d < kTiles; d++) o[t][d] *= f;
                    }
                }
                const float down = as_float((254u << 23) - bits_of(ev[t]));
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= down;
            }
            M::split(x, p[t]);
        }
    }

    // o += p times the block's values; value(tile): the operand of 16 channels.
    template <class Value>
    __device__ __forceinline__ void products(const u32x4 (&p)[kCols][M::kParts], Value value) {
#pragma unroll
        for (int d = 0; d < kTiles; d += 2) {
            const u32x4 a = value(d), b = value(d + 1);
#pragma unroll
            for (int k = 0; k < M::kParts; k++)
#pragma unroll
                for (int t = 0; t < kCols; t++) {
                    o[t][d] = M::mfma(a, p[t][k], o[t][d]);
                    o[t][d + 1] = M::mfma(b, p[t][k], o[t][d + 1]);
                }
        }
    }

    // Notes which columns see values that are not finite: ones in their places times ones for the tokens seen.
    template <class Value>
    __device__ __forceinline__ void note_bad(int first, Value value) {
        constexpr uint32_t kOne = kType == kKvBf16 ? 0x3f80u : 0x3c00u;
        const int mine = first + ((threadIdx.x >> 4) & 3) * 4;
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            u32x4 seen = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int j = mine + (i >> 2) * 16 + (i & 3);
                seen[i >> 1] |= j <= lim[t] && j >= low[t] ? kOne << (16 * (i & 1)) : 0u;
            }
            uint64_t found = 0;
#pragma unroll 1
            for (int d = 0; d < kTiles; d++) {
                u32x4 a = not_finite<kType>(value(d));
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = (a[i] >> 15) * kOne;
                const f32x4 n = M::mfma(a, seen, f32x4{0, 0, 0, 0});
#pragma unroll
                for (int i = 0; i < 4; i++) found |= (uint64_t)(n[i] > 0.0f) << (4 * d + i);
            }
            bad[t][0] |= (uint32_t)found;
            bad[t][1] |= (uint32_t)(found >> 32);
        }
    }

    // After the last block: l over the column's lanes, NaN where bad values were noted.
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            l[t] = column_sum(l[t]);
            if constexpr (kType != kKvI8) {
                if (__ballot((bad[t][0] | bad[t][1]) != 0)) {
#pragma unroll
                    for (int d = 0; d < kTiles; d++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[t][d][i] = bad[t][d >> 3] >> ((4 * d + i) & 31) & 1 ? __builtin_nanf("") : o[t][d][i];
                }
            }
        }
    }
    // Column t's four channels 16 d + 4 (lane / 16) .. + 3, times f, which is no more than one over the column's sum.
    __device__ __forceinline__ f32x4 output(int t, int d, float f) const {
        f32x4 y = o[t][d] * f;
        if constexpr (kType == kKvI8) y *= ev[t];
        return y;
    }
};
// One over a sum of probabilities; a row that sees nothing has 0 and gives zeros.
__device__ __forceinline__ float one_over(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// Key operands of a block's bytes, read through `load(byte)` (16 of them, this lane's), and value operands.
template <int kType, int kDp, class Load>
__device__ __forceinline__ u32x4 key_operand(int tile, int chunk, Load load) {
    if constexpr (kType == kKvI8) {
        const u32x4 w = load((tile * (kDp / 64) + (chunk >> 1)) * 1024);
        return chunk & 1 ? widened(w.z, w.w) : widened(w.x, w.y);
    } else {
        return load((tile * (kDp / 32) + chunk) * 1024);
    }
}
template <int kType, int kDp, class Load>
__device__ __forceinline__ u32x4 value_operand(int tile, Load load) {
    constexpr int kBase = kv_plane_bytes(kType, kDp);
    if constexpr (kType == kKvI8) {
        const u32x4 w = load(kBase + (tile >> 1) * 1024);
        return tile & 1 ? widened(w.z, w.w) : widened(w.x, w.y);
    } else {
        return load(kBase + tile * 1024);
    }
}

// The first token that a row at `last` sees; before the first token it sees none, whatever this says.
__device__ __forceinline__ int first_seen(int last, int window) { return window ? max(max(last, 0) - window + 1, 0) : 0; }

// How a launch cuts its work. A request of `least` to `most` columns has tiles of `cols` columns (2^cols_log2), and a tile's blocks are
// cut into pieces of the same size, none of fewer blocks than least_blocks. `target` is the number of workgroups that the chip holds at
// a time, for each key head. Fewer tiles are cut into the smallest pieces that still are no more than that: a workgroup more is a round
// more (64 decode rows of 1 k to 8 k tokens in 512 workgroups 221 us, 1072 pieces of one size and their remainders 238;
// 60 drafted rows over 24 k in 8 bits 95 and 107).
// More tiles than that stay whole, but for those longer than `slack` times what a workgroup has on average, and if there are none go by
// the place of their last column, the last ones (with the longest spans) first.
struct Cut {
    int cols_log2, least, most, target, least_blocks;
    float slack;
    int window, group;
    int slots, tiles;  // most of a key head's partial outputs, and of its tiles
    int planned;       // the requests' items are counted by a launch of their own (AttendArgs::plan holds them)
};
// A launch's tiles that the join has to look at (none if all are whole), and where the items were counted before: one over a piece's
// size, and the items, tiles and slots of each 64 requests.
struct CutPlan {
    int joins, tiles;
    float inv;
    int unused;
};
struct CutChunk {
    int items, tiles, slots, unused;
};
// What the join needs to know of a tile, written by the tile's first piece.
struct TilePlan {
    int first_row, rows, col0;
    int pieces, slot;  // slot: the first piece's place among the head's partial outputs
};
struct TileWork : TilePlan {
    int r, tile, piece;
    int tile_index;      // among all requests' tiles
    int place;           // of the request's first new token
    int block0, block1;  // the piece's blocks
};

// A lane's request.
struct CutRequest {
    int first, n, place, tiles, blocks;  // blocks: of its longest tile, at most
    float sum;                           // of its tiles' blocks, about
};
// Pieces of a tile of so many blocks, `inv` being one over a piece's most, give or take a thousandth: their sizes follow from the number.
__device__ __forceinline__ int cut_pieces(int blocks, float inv) { return max((int)ceilf(fmaf((float)blocks, inv, -1.0e-3f)), 1); }
// Blocks that the tokens place + i0 .. place + i1 see: [x, y).
__device__ __forceinline__ int2 cut_blocks(const Cut& c, const KvPool& pool, const KvBatch& b, int place, int i0, int i1) {
    const int64_t last = min((int64_t)place + i1, (int64_t)b.width * pool.page - 1);
    const int64_t first = c.window ? max((int64_t)place + i0 - c.window + 1, (int64_t)0) : 0;
    const int x = (int)(first / kKvBlock);
    return make_int2(x, last < first ? x : (int)(last / kKvBlock) + 1);
}
__device__ __forceinline__ CutRequest cut_load(const Cut& c, const KvPool& pool, const KvBatch& b, int r) {
    CutRequest q{0, 0, 0, 0, 0, 0.0f};
    if (r >= b.requests) return q;
    const KvRows m = kv_rows(b, r);
    const int len = kv_length(b, r), cols = m.n * c.group;
    if (!m.n || cols < c.least || cols > c.most) return q;
    q.first = m.first;
    q.n = m.n;
    q.place = len - m.n;
    q.tiles = ((cols - 1) >> c.cols_log2) + 1;
    const int2 s = cut_blocks(c, pool, b, q.place, 0, m.n - 1);
    const int all = s.y - s.x, rows = min((1 << c.cols_log2) / c.group + 2, m.n);  // a tile's rows, at most
    q.blocks = c.window ? min(all, (int)(((int64_t)c.window + rows) / kKvBlock) + 2) : all;
    const int2 f = cut_blocks(c, pool, b, q.place, 0, min(rows, m.n) - 1);
    q.sum = (float)q.tiles * (c.window ? (float)q.blocks : 0.5f * (float)(q.blocks + f.y - f.x));
    return q;
}

// Blocks of a piece, from all requests' sum of blocks and number of tiles, before it is fitted to the number of workgroups.
__device__ __forceinline__ float cut_piece(const Cut& c, float sum, int tiles) {
    return fmaxf(ceilf(sum / (float)c.target * (tiles >= c.target ? c.slack : 1.0f)), (float)c.least_blocks);
}
// A request's items, its tiles taken as long as the longest of them, and its slots: whole tiles have none.
__device__ __forceinline__ int2 cut_items(const CutRequest& q, float inv) {
    const int items = q.tiles * cut_pieces(q.blocks, inv);
    return make_int2(items, items > q.tiles ? items : 0);
}

// Of lanes with `tiles` tiles from `place` on, the tile number `item` by the place of its last column, the last one first: its lane, and
// its number there. There are more than `item` of them.
__device__ __forceinline__ int cut_latest(const Cut& c, int place, int tiles, int item, int& tile) {
    // x: the largest number that no more than `item` tiles end past (base + tile: a tile's end, in tiles)
    const int base = (int)min(max(((int64_t)place * c.group) >> c.cols_log2, (int64_t)0), (int64_t)1 << 30);
    int lo = -1, hi = tiles ? base + tiles : 0;
    hi = wave_max(hi);  // none past hi; more than `item` past lo
    int past = 0;
    while (hi - lo > 1) {
        const int x = lo + (hi - lo) / 2;
        const int n = wave_sum(min(max(base + tiles - 1 - x, 0), tiles));
        if (n <= item) {
            hi = x;
            past = n;
        } else {
            lo = x;
        }
    }
    const int at = hi - base;  // the tile that ends there
    uint64_t votes = __ballot(at >= 0 && at < tiles);
    for (int i = past; i < item; i++) votes &= votes - 1;
    const int l = __ffsll((unsigned long long)votes) - 1;
    tile = __builtin_amdgcn_readlane(at, l);
    return l;
}

// The same for up to 64 requests of many tiles each, whose spans differ: every tile has as many pieces as its own span gives, tiles of
// the most pieces come first, whole ones last, the longest of them first. (Counting each tile as the longest of its request, 2048 prompt
// rows of 32 query heads over 8 took 119 us, so 95: the items of no work between the others kept workgroups out for 50.)
__device__ __forceinline__ bool cut_tiles(const Cut& c, const KvPool& pool, const KvBatch& b, CutPlan* plan, int item, TileWork& w) {
    const CutRequest q = cut_load(c, pool, b, threadIdx.x & 63);
    const int tiles = wave_sum(q.tiles), longest = wave_max(q.blocks);
    // the request's blocks of tile u, and its first tile of more than x blocks
    auto span = [&](int u) {
        const int last = q.place + min(q.n - 1, (((u + 1) << c.cols_log2) - 1) / c.group);
        return last < 0 ? 0 : min(last / kKvBlock + 1, q.blocks);
    };
    auto above = [&](int x) {
        if (x >= q.blocks) return q.tiles;
        const int row = x * kKvBlock - q.place;
        return row <= 0 ? 0 : min((row * c.group) >> c.cols_log2, q.tiles - 1);
    };
    int piece = uniform((int)cut_piece(c, wave_sum(q.sum), tiles));
    if (tiles < c.target && longest > piece) {
        // halving what lies between the mean, which may give too many, and the longest tile
        const int most = wave_max(q.tiles);
        auto items = [&](int size) {
            const int layers = uniform((longest + size - 1) / size);
            int n = 0;
            if (most < layers) {
                for (int u = 0; u < most; u++) n += u < q.tiles ? max((span(u) + size - 1) / size, 1) : 0;
            } else {
                n = q.tiles;
                for (int k = 1; k < layers; k++) n += q.tiles - above(k * size);
            }
            return wave_sum(n);
        };
        int over = piece;
        if (items(piece) > c.target) {
            piece = longest;
            for (int i = 0; i < 5 && piece - over > 1; i++) {
                const int half = (piece + over) >> 1;
                if (items(half) > c.target)
                    over = half;
                else
                    piece = half;
            }
        }
    }
    const bool fit = tiles <= c.tiles;  // (if not, offsets overlap: none of the call's tiles)
    if (blockIdx.x == 0) {
        const int joins = wave_sum(q.tiles - above(piece));
        if (threadIdx.x == 0) plan->joins = fit ? joins : 0;
    }
    if (!fit) return false;
    int left = q.tiles, l = -1;
    w.slot = w.tile_index = w.piece = 0;
    w.pieces = 1;
    while (longest > piece) {
        const int mine = left ? (span(left - 1) + piece - 1) / piece : 0, most = wave_max(mine);
        if (most < 2) break;
        const int low = mine == most ? min(above((most - 1) * piece), left - 1) : left, n = left - low, upto = wave_upto(n);
        const int all = __builtin_amdgcn_readlane(upto, 63);
        if (item < all * most) {
            const int nth = uniform(item / most);
            l = __ffsll((unsigned long long)__ballot(upto > nth)) - 1;
            w.pieces = most;
            w.piece = item - nth * most;
            w.tile = __builtin_amdgcn_readlane(left, l) - 1 - (nth - __builtin_amdgcn_readlane(upto - n, l));
            w.slot += nth * most;
            w.tile_index += nth;
            break;
        }
        item -= all * most;
        w.slot += all * most;
        w.tile_index += all;
        left = low;
    }
    if (l < 0) {
        if (item >= wave_sum(left)) return false;
        l = cut_latest(c, q.place, left, item, w.tile);
        w.tile_index += item;
    }
    w.r = l;
    w.first_row = __builtin_amdgcn_readlane(q.first, l);
    w.rows = __builtin_amdgcn_readlane(q.n, l);
    w.place = __builtin_amdgcn_readlane(q.place, l);
    w.col0 = w.tile << c.cols_log2;
    const int2 s = cut_blocks(c, pool, b, w.place, uniform(w.col0 / c.group), uniform(min(w.rows - 1, (w.col0 + (1 << c.cols_log2) - 1) / c.group)));
    const int size = uniform((s.y - s.x + w.pieces - 1) / w.pieces);
    w.block0 = min(s.x + w.piece * size, s.y);
    w.block1 = min(w.block0 + size, s.y);
    return w.pieces == 1 || w.slot + w.pieces <= c.slots;
}

// Item `item` of a key head; false past the last one. Every wave finds it for itself: lanes hold 64 requests at a time, or in a planned
// launch 64 times 64 of them and then the item's.
__device__ __forceinline__ bool cut_item(const Cut& c, const KvPool& pool, const KvBatch& b, CutPlan* plan, int item, TileWork& w) {
    const int lane = threadIdx.x & 63;
    CutRequest q;
    float inv;
    int tiles = 0, longest = 0;
    if (c.planned) {
        if (!uniform(plan->tiles)) return false;
        inv = as_float((uint32_t)uniform((int)__builtin_bit_cast(uint32_t, plan->inv)));
    } else {
        q = cut_load(c, pool, b, lane);
        float sum = q.sum;
        tiles = q.tiles, longest = q.blocks;
        for (int base = 64; base < b.requests; base += 64) {
            const CutRequest o = cut_load(c, pool, b, base + lane);
            sum += o.sum;
            tiles += o.tiles;
            longest = max(longest, o.blocks);
        }
        sum = wave_sum(sum);
        tiles = wave_sum(tiles);
        longest = wave_max(longest);
        float piece = cut_piece(c, sum, tiles);
        if (tiles < c.target && b.requests <= 64 && (float)longest > piece) {
            // halving what lies between the mean, which may give too many, and the longest tile
            float over = piece;
            if (wave_sum(cut_items(q, 1.0f / piece).x) > c.target) {
                piece = (float)longest;
                for (int i = 0; i < 5 && piece - over > 1.0f; i++) {
                    const float half = floorf(0.5f * (piece + over));
                    if (wave_sum(cut_items(q, 1.0f / half).x) > c.target)
                        over = half;
                    else
                        piece = half;
                }
            }
        }
        inv = as_float((uint32_t)uniform((int)__builtin_bit_cast(uint32_t, 1.0f / piece)));
        const bool fit = tiles <= c.tiles;  // (if not, offsets overlap: none of the call's tiles)
        if (blockIdx.x == 0 && threadIdx.x == 0) plan->joins = fit && cut_pieces(longest, inv) > 1 ? tiles : 0;
        if (!fit) return false;
    }
    int l = 0, before = 0, tiles_before = 0, slots_before = 0;
    w.piece = 0;
    w.r = 0;
    if (!c.planned && b.requests <= 64 && cut_pieces(longest, inv) == 1) {
        if (item >= tiles) return false;
        l = cut_latest(c, q.place, q.tiles, item, w.tile);
        w.r = l;
        w.slot = 0;
        w.tile_index = item;
    } else {
        // of 64 sums at a time (a lane's items, tiles and slots) the one that `item` falls into
        auto found = [&](int items, int its_tiles, int slots) {
            const int upto = wave_upto(items), tiles_upto = wave_upto(its_tiles), slots_upto = wave_upto(slots);
            const int all = __builtin_amdgcn_readlane(upto, 63);
            if (item >= before + all) {
                before += all;
                tiles_before += __builtin_amdgcn_readlane(tiles_upto, 63);
                slots_before += __builtin_amdgcn_readlane(slots_upto, 63);
                return false;
            }
            l = __ffsll((unsigned long long)__ballot(before + upto > item)) - 1;
            before += __builtin_amdgcn_readlane(upto - items, l);
            tiles_before += __builtin_amdgcn_readlane(tiles_upto - its_tiles, l);
            slots_before += __builtin_amdgcn_readlane(slots_upto - slots, l);
            return true;
        };
        int first = 0;
        if (c.planned) {
            const CutChunk* chunks = (const CutChunk*)(plan + 1);
            const int count = (b.requests + 63) >> 6;
            for (int base = 0;; base += 64) {
                if (base >= count) return false;
                const CutChunk s = base + lane < count ? chunks[base + lane] : CutChunk{0, 0, 0, 0};
                if (found(s.items, s.tiles, s.slots)) {
                    first = 64 * (base + l);
                    break;
                }
            }
            q = cut_load(c, pool, b, first + lane);
        }
        for (;; first += 64) {
            if (first >= b.requests) return false;
            if (first && !c.planned) q = cut_load(c, pool, b, first + lane);
            const int2 mine = cut_items(q, inv);
            if (found(mine.x, q.tiles, mine.y)) break;
            if (c.planned) return false;
        }
        w.r = first + l;
        const int pieces = uniform(cut_pieces(__builtin_amdgcn_readlane(q.blocks, l), inv));
        const int nth = uniform((item - before) / pieces);
        w.piece = item - before - nth * pieces;
        w.tile = __builtin_amdgcn_readlane(q.tiles, l) - 1 - nth;
        w.slot = slots_before + nth * pieces;
        w.tile_index = tiles_before + nth;
    }
    w.first_row = __builtin_amdgcn_readlane(q.first, l);
    w.rows = __builtin_amdgcn_readlane(q.n, l);
    w.place = __builtin_amdgcn_readlane(q.place, l);
    w.col0 = w.tile << c.cols_log2;
    const int2 s = cut_blocks(c, pool, b, w.place, uniform(w.col0 / c.group), uniform(min(w.rows - 1, (w.col0 + (1 << c.cols_log2) - 1) / c.group)));
    w.pieces = uniform(cut_pieces(s.y - s.x, inv));
    const int size = w.pieces == 1 ? s.y - s.x : (uniform((s.y - s.x + w.pieces - 1) / w.pieces) + 3) & ~3;  // (whole turns of four waves)
    w.block0 = min(s.x + w.piece * size, s.y);
    w.block1 = min(w.block0 + size, s.y);
    if (w.slot + w.pieces > c.slots && w.pieces > 1) return false;
    return w.piece < w.pieces;
}
// A walk over blocks first, first + step, ..: their pages in 64 lanes at a time.
struct BlockWalk {
    const int* table;  // the request's
    int step, entries, pages, shift;  // shift: log2 of a page's blocks
    int first, held;
    __device__ __forceinline__ void start(const KvPool& p, const int* row, int width, int block, int stride) {
        table = row;
        entries = width;
        pages = p.pages;
        shift = 31 - __builtin_clz(p.page / kKvBlock);
        step = stride;
        first = block;
        fetch();
    }
    __device__ __forceinline__ void fetch() {
        const int64_t entry = ((int64_t)first + (int64_t)(threadIdx.x & 63) * step) >> shift;
        const int p = table[min(entry, (int64_t)entries - 1)];
        held = entry < entries && p >= 0 && p < pages ? p : -1;
    }
    // Page of block first + i * step, i rising by one from call to call, or -1.
    __device__ __forceinline__ int page(int i) {
        if (i && (i & 63) == 0) {
            first += 64 * step;
            fetch();
        }
        return __builtin_amdgcn_readlane(held, i & 63);
    }
};

// Partial outputs of a piece: for each 16-column tile `ml` [16] references and [16] sums, and the outputs of the piece alone, divided by
// its sums, as the lanes hold them.
__host__ __device__ constexpr int part_floats(int cols, int dp) { return cols * (dp + 2); }

}  // namespace ovfq
