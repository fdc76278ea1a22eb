// attend.h — what the attention kernels over a paged cache share: their arithmetic on one block of 32 tokens, and the way the work
// is cut.
//
//   out = softmax(scale q . k) v   over the tokens j with  position - window < j <= position  (window 0: all up to the position)
//
// A kernel's columns are (row, query head) pairs of one request and key head, row by row: column c is row c / group, head c % group.
// Products are MFMA 16x16x32 with the cache's operands as the first factor, so that a lane's results belong to one column (lane % 16)
// and to the tokens whose values the same lane group loads for the second product: probabilities never change lanes.
//
// Rounding. q and p are fp32 and enter the products in parts that carry all of fp32's bits but the last two at most: two fp16 parts
// beside fp16 and int8 operands (22 bits), three bf16 parts beside bf16 ones (24). q is scaled by a power of two to below 2 for that;
// p is 2^10 at the largest score that its column has met when it last moved its reference, which it does when a score passes that by
// 2^4, so fp16 has 2^24 below the largest p and no overflow above. Sums and references are fp32. int8 operands are widened to fp16,
// which is exact; a token's key scale multiplies its scores, its value scale its probabilities, against a power of two kept for the
// column.
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

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTop = 10.0f, kRoom = 4.0f;  // log2 of p at a new reference, and how far it may grow before the next

template <int kType>
struct KvMath {
    static constexpr int kParts = kType == kKvBf16 ? 3 : 2;
    static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
        if constexpr (kType == kKvBf16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    }
    // Eight fp32 values as kParts operands that add up to them.
    static __device__ __forceinline__ void split(const float (&x)[8], u32x4 (&part)[kParts]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f32x2 v = {x[2 * i], x[2 * i + 1]};
#pragma unroll
            for (int p = 0; p < kParts; p++) {
                uint32_t w;
                f32x2 back;
                if constexpr (kType == kKvBf16) {
                    w = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b16x2));
                    back = f32x2{as_float(w << 16), as_float(w & 0xffff0000u)};
                } else {
                    const h16x2 h = __builtin_convertvector(v, h16x2);
                    w = __builtin_bit_cast(uint32_t, h);
                    back = __builtin_convertvector(h, f32x2);
                }
                part[p][i] = w;
                if (p + 1 < kParts) {
                    v.x = v.x - back.x;
                    v.y = v.y - back.y;
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
    float ev[kCols];             // int8: the power of two that value scales are divided by, 0 at first
    uint32_t bad[kCols][2];      // bit 4 d + i: the column sees a value that is not finite in o[][d][i]'s channel (of masked blocks)

    // Column `col` of the tile has query row x (NULL: none) and sees the tokens [first, last].
    __device__ __forceinline__ void column(int t, const float* x, int dim, float scale, int first, int last) {
        const int g = (threadIdx.x >> 4) & 3;
        float v[kChunks][8];
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            const int d = c * 32 + g * 8;
            f32x4u a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (x && d < dim) {
                a = *(const f32x4u*)(x + d);
                b = *(const f32x4u*)(x + d + 4);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[c][i] = (i < 4 ? a[i & 3] : b[i & 3]) * scale;
                top = fmaxf(top, fabsf(v[c][i]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
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
        lim[t] = x ? last : -1;
        low[t] = first;
        ref[t] = -kInf;
        l[t] = 0.0f;
        ev[t] = 0.0f;
        bad[t][0] = bad[t][1] = 0;
#pragma unroll
        for (int d = 0; d < kTiles; d++) o[t][d] = f32x4{0, 0, 0, 0};
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

    // Scores into probabilities, split for the second product. first: the block's first token; ks, vs: int8's scales of this lane's tokens.
    __device__ __forceinline__ void probabilities(f32x4 (&s)[kCols][2], u32x4 (&p)[kCols][M::kParts], bool masked, int first,
                                                  const f32x4 (&ks)[2], const f32x4 (&vs)[2]) {
        const int mine = first + ((threadIdx.x >> 4) & 3) * 4;
        bool move = false;
        float top[kCols], vtop[kCols];
#pragma unroll
        for (int t = 0; t < kCols; t++) {
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[t][h][i] *= qs[t];
                    if constexpr (kType == kKvI8) s[t][h][i] *= ks[h][i];
                }
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < kCols; t++) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = mine + 16 * h + i;
                        s[t][h][i] = (int)(j <= lim[t]) & (int)(j >= low[t]) ? s[t][h][i] : -kInf;
                    }
            }
        }
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            top[t] = -kInf;
            vtop[t] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    top[t] = fmaxf(top[t], s[t][h][i]);
                    // (a hidden token's scale counts for nothing)
                    if constexpr (kType == kKvI8) vtop[t] = fmaxf(vtop[t], masked && s[t][h][i] == -kInf ? 0.0f : vs[h][i]);
                }
            move = move | (top[t] > ref[t] + kTop + kRoom);
            if constexpr (kType == kKvI8) move = move | (vtop[t] > ev[t]);
        }
        if (__ballot(move)) {
#pragma unroll
            for (int t = 0; t < kCols; t++) {
                float m = fmaxf(top[t], __shfl_xor(top[t], 16, 64));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                float f = 1.0f;
                if (m > ref[t] + kTop + kRoom) {
                    f = __builtin_amdgcn_exp2f(ref[t] - (m - kTop));
                    ref[t] = m - kTop;
                    l[t] *= f;
                }
                if constexpr (kType == kKvI8) {
                    float v = fmaxf(vtop[t], __shfl_xor(vtop[t], 16, 64));
                    v = fmaxf(v, __shfl_xor(v, 32, 64));
                    if (v > ev[t]) {
                        const uint32_t e = min((__builtin_bit_cast(uint32_t, v) >> 23) + 1u, 253u);
                        f *= ev[t] * as_float((254u - e) << 23);
                        ev[t] = as_float(e << 23);
                    }
                }
#pragma unroll
                for (int d = 0; d < kTiles; d++) o[t][d] *= f;
            }
        }
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            const float r = ref[t] == -kInf ? 0.0f : ref[t];
            float x[8];
            float down = 0.0f;
            if constexpr (kType == kKvI8) down = ev[t] > 0.0f ? as_float((254u << 23) - __builtin_bit_cast(uint32_t, ev[t])) : 0.0f;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = __builtin_amdgcn_exp2f(s[t][h][i] - r);
                    l[t] += v;
                    x[4 * h + i] = v;
                    if constexpr (kType == kKvI8) {
                        const float w = v * (vs[h][i] * down);
                        x[4 * h + i] = masked && s[t][h][i] == -kInf ? 0.0f : w;
                    }
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
    template <int kUnrollNotes, class Value>
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
#pragma unroll kUnrollNotes
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

    // After the last block: l over the column's lanes, int8's power of two back into o, NaN where bad values were noted.
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            l[t] += __shfl_xor(l[t], 16, 64);
            l[t] += __shfl_xor(l[t], 32, 64);
            if constexpr (kType == kKvI8) {
#pragma unroll
                for (int d = 0; d < kTiles; d++) o[t][d] *= ev[t];
            } else if (__ballot((bad[t][0] | bad[t][1]) != 0)) {
#pragma unroll
                for (int d = 0; d < kTiles; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[t][d][i] = bad[t][d >> 3] >> ((4 * d + i) & 31) & 1 ? __builtin_nanf("") : o[t][d][i];
            }
        }
    }
};

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

// How a launch cuts its work: tiles of `cols` columns, each tile's blocks in pieces of so many that all tiles of one key head give
// about `target` pieces (whole tiles where !split). Which requests: those of `least` to `most` columns.
struct Cut {
    int cols, least, most, target, least_blocks;
    bool split;
    int window, group;
    int slots;  // of a key head's partial outputs (offsets that overlap could ask for more: those pieces are left out)
};
struct TileWork {
    int r, tile, piece, slot;  // slot: the piece's place among the head's partial outputs
    int first_row, rows;       // the request's
    int place;                 // of its first new token
    int col0;                  // the tile's first column
    int block0, block1;        // the piece's blocks
    int pieces;                // of the tile
    int pieces_of_request;     // slots that each of its tiles has
};

__device__ __forceinline__ int cut_tiles(const Cut& c, int n) {
    const int cols = n * c.group;
    return n && cols >= c.least && cols <= c.most ? (cols + c.cols - 1) / c.cols : 0;
}
// Blocks that the rows i0 .. i1 of a request see: [x, y).
__device__ __forceinline__ int2 cut_blocks(const Cut& c, const KvPool& pool, const KvBatch& b, int place, int i0, int i1) {
    const int64_t last = min((int64_t)place + i1, (int64_t)b.width * pool.page - 1);
    const int64_t first = c.window ? max((int64_t)place + i0 - c.window + 1, (int64_t)0) : 0;
    const int x = (int)(first / kKvBlock);
    return make_int2(x, last < first ? x : (int)(last / kKvBlock) + 1);
}
__device__ __forceinline__ int cut_request_blocks(const Cut& c, const KvPool& pool, const KvBatch& b, int r, int n) {
    const int2 s = cut_blocks(c, pool, b, kv_length(b, r) - n, 0, n - 1);
    return s.y - s.x;
}
// Blocks a piece.
__device__ __forceinline__ int cut_piece(const Cut& c, const KvPool& pool, const KvBatch& b) {
    if (!c.split) return 0x7fffffff;
    float all = 0.0f;
    for (int r = threadIdx.x & 63; r < b.requests; r += 64) {
        const int n = kv_rows(b, r).n, tiles = cut_tiles(c, n);
        if (tiles) all += (float)tiles * (float)cut_request_blocks(c, pool, b, r, n);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) all += __shfl_xor(all, off, 64);
    return uniform(max((int)fminf(ceilf(all / (float)c.target), 1.0e9f), c.least_blocks));
}
__device__ __forceinline__ int cut_pieces(int blocks, int piece) { return blocks > piece ? (blocks + piece - 1) / piece : 1; }

// A request's tile and its piece, or false where it has no such piece.
__device__ __forceinline__ bool cut_tile(const Cut& c, const KvPool& pool, const KvBatch& b, int piece, int r, int tile, int j,
                                         int before, TileWork& w) {
    KvRows m = kv_rows(b, r);
    m.first = uniform(m.first);
    m.n = uniform(m.n);
    w.r = r;
    w.tile = tile;
    w.piece = j;
    w.first_row = m.first;
    w.rows = m.n;
    w.place = uniform(kv_length(b, r)) - m.n;
    w.col0 = tile * c.cols;
    w.pieces_of_request = uniform(cut_pieces(cut_request_blocks(c, pool, b, r, m.n), piece));
    w.slot = before + tile * w.pieces_of_request + j;
    const int2 s = cut_blocks(c, pool, b, w.place, w.col0 / c.group, min(m.n - 1, (w.col0 + c.cols - 1) / c.group));
    w.pieces = cut_pieces(s.y - s.x, piece);
    w.block0 = s.x + j * min(piece, s.y - s.x);
    w.block1 = s.y - w.block0 > piece ? w.block0 + piece : s.y;
    return j < w.pieces && (w.pieces == 1 || w.slot - j + w.pieces <= c.slots);
}
// Item `item` of a key head: the pieces of its requests' tiles, the last tiles (with the longest spans) first.
__device__ __forceinline__ bool cut_item(const Cut& c, const KvPool& pool, const KvBatch& b, int item, TileWork& w) {
    const int piece = cut_piece(c, pool, b);
    int r = 0, before = 0;
    const bool any = kv_find(b.requests, item, r, before, [&](int q) {
        const int n = kv_rows(b, q).n, tiles = cut_tiles(c, n);
        return tiles ? tiles * cut_pieces(cut_request_blocks(c, pool, b, q, n), piece) : 0;
    });
    if (!any) return false;
    const int n = uniform(kv_rows(b, r).n), each = uniform(cut_pieces(cut_request_blocks(c, pool, b, r, n), piece));
    return cut_tile(c, pool, b, piece, r, cut_tiles(c, n) - 1 - item / each, item % each, before, w);
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
        const int p = entry < entries ? table[entry] : -1;
        held = p >= 0 && p < pages ? p : -1;
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

// Partial outputs of a piece: for each 16-column tile `ml` [16] references and [16] sums, and o as the lanes hold it.
__host__ __device__ constexpr int part_floats(int cols, int dp) { return cols * (dp + 2); }

}  // namespace ovfq
