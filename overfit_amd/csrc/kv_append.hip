// kv_append.hip — new tokens into a paged cache: their keys turned by their positions and rounded to the cache's type, their values
// beside them, their queries turned by the same angles.
//   (a, b) -> (a c - b s, b c + a s) for pair j of a head, c and s = scale * cos and sin of position[axis_j] * freq_j
// The pairs are neighbours (2 j, 2 j + 1) or halves (j, j + rotary / 2); channels past `rotary` stay.
//
// Angles are taken in turns in fp64, with the rounding errors of both products (position * freq has up to 55 bits) carried along, so a
// position of 2^31 has the same 2^-50 as a near one, and cos and sin come from polynomials of the remainder (10^-13 off); both are
// rounded to fp32 once. Products and sums of
// the rotation are single fp32 operations; the rounding to the cache's type is the only other one, half a step of that type.
//
// Bound: HBM for many rows (each fp32 row is read once, written once), the launch and three dependent reads (offsets and length, page,
// rows) for one. Queries and keys have a workgroup a row, four for batches below the chip's workgroups, which share the row's heads;
// values one for a share of a block of the cache. (us, 1 / 1297 / 4096 rows of 32 and 8 heads of 128: 4.1 / 13.6 / 42.5; a copy of the bytes 0.01 / 11.4
// / 36.1.)
#include "kv_cache.h"

namespace ovfq {

int kv_padded_dim(int type, int dim) {
    if (dim <= 64) return 64;
    if (dim <= 96 && type != kKvI8) return 96;
    return dim <= 128 ? 128 : 256;
}
size_t kv_block_bytes(int type, int dp) { return (size_t)kv_bytes(type, dp); }

namespace {

// Planes are aligned to four bytes only.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMaxPairs = 128;

struct Turn {
    float c, s;
};
__device__ Turn turn_of(int position, float freq, float scale) {
    const double a = (double)position * (double)freq, low = fma((double)position, (double)freq, -a);
    const double kInv = 0.15915494309189535, kInvLow = -9.839338337591243e-18;  // 1 / (2 pi) in two parts
    const double t = a * kInv;
    const double rest = fma(a, kInv, -t) + fma(a, kInvLow, low * kInv);
    double f = (t - rint(t)) + rest;  // in turns, [-1/2, 1/2]
    const double quarter = rint(f * 4.0);
    const double x = (f - quarter * 0.25) * 6.283185307179586;  // [-pi / 4, pi / 4]
    const double z = x * x;
    double s = fma(z, 1.6059043836821613e-10, -2.505210838544172e-8);
    s = fma(z, s, 2.7557319223985893e-6);
    s = fma(z, s, -1.984126984126984e-4);
    s = fma(z, s, 8.333333333333333e-3);
    s = fma(z, s, -1.6666666666666666e-1);
    s = fma(z * x, s, x);
    double c = fma(z, -1.1470745597729725e-11, 2.08767569878681e-9);
    c = fma(z, c, -2.7557319223985888e-7);
    c = fma(z, c, 2.48015873015873e-5);
    c = fma(z, c, -1.388888888888889e-3);
    c = fma(z, c, 4.1666666666666664e-2);
    c = fma(z, c, -0.5);
    c = fma(z, c, 1.0);
    const int n = (int)quarter & 3;
    const double cc = n & 1 ? s : c, ss = n & 1 ? c : s;
    const double m = (double)scale;
    return Turn{(float)((n == 1 || n == 2 ? -cc : cc) * m), (float)((n >= 2 ? -ss : ss) * m)};
}

// Eight channels d .. d + 7 of a head's row x, rotated. kFast: pairs and halves never part within four channels.
template <bool kFast>
__device__ __forceinline__ void rotated8(const float* __restrict__ x, int d, const KvRope& r, const float* cs, float (&o)[8]) {
    if constexpr (kFast) {
        const f32x4u a = *(const f32x4u*)(x + d), b = *(const f32x4u*)(x + d + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[i] = a[i];
            o[4 + i] = b[i];
        }
        if (d >= r.rotary) return;
        if (!r.halves) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float c = cs[d / 2 + i], s = cs[kMaxPairs + d / 2 + i], p = o[2 * i], q = o[2 * i + 1];
                o[2 * i] = p * c - q * s;
                o[2 * i + 1] = q * c + p * s;
            }
            return;
        }
        const int half = r.rotary >> 1;
        const bool second = d >= half;
        const int j = second ? d - half : d;
        const float* other = x + (second ? d - half : d + half);
        const f32x4u e = *(const f32x4u*)other, f = *(const f32x4u*)(other + 4);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float c = cs[j + i], s = cs[kMaxPairs + j + i], y = i < 4 ? e[i & 3] : f[i & 3];
            o[i] = second ? o[i] * c + y * s : o[i] * c - y * s;
        }
    } else {
        const int half = r.rotary >> 1;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int e = d + i;
            float v = x[e];
            if (e < r.rotary) {
                const int j = r.halves ? (e < half ? e : e - half) : e >> 1;
                const bool second = r.halves ? e >= half : (e & 1);
                const float y = x[r.halves ? (second ? e - half : e + half) : e ^ 1], c = cs[j], s = cs[kMaxPairs + j];
                v = second ? v * c + y * s : v * c - y * s;
            }
            o[i] = v;
        }
    }
}

// One unit of a query row: four pairs (or what is left of them), or four channels behind the rotated ones. Pairs stay with one thread,
// so q_out may be q.
template <bool kFast>
__device__ __forceinline__ void rotate_query(const float* x, float* y, int dim, int unit, const KvRope& r, const float* cs) {
    const int half = r.rotary >> 1, pair_units = (half + 3) >> 2;
    if (unit >= pair_units) {
        if (x == y) return;
        const int d = r.rotary + 4 * (unit - pair_units);
        if (kFast) {
            *(f32x4u*)(y + d) = *(const f32x4u*)(x + d);
        } else {
            for (int i = d; i < dim && i < d + 4; i++) y[i] = x[i];
        }
        return;
    }
    const int j = 4 * unit;
    if constexpr (kFast) {
        const f32x4u c = *(const f32x4u*)(cs + j), s = *(const f32x4u*)(cs + kMaxPairs + j);
        if (r.halves) {
            const f32x4u a = *(const f32x4u*)(x + j), b = *(const f32x4u*)(x + half + j);
            *(f32x4u*)(y + j) = a * c - b * s;
            *(f32x4u*)(y + half + j) = b * c + a * s;
        } else {
            f32x4u a = *(const f32x4u*)(x + 2 * j), b = *(const f32x4u*)(x + 2 * j + 4);
            *(f32x4u*)(y + 2 * j) = f32x4u{a.x * c.x - a.y * s.x, a.y * c.x + a.x * s.x, a.z * c.y - a.w * s.y, a.w * c.y + a.z * s.y};
            *(f32x4u*)(y + 2 * j + 4) =
                f32x4u{b.x * c.z - b.y * s.z, b.y * c.z + b.x * s.z, b.z * c.w - b.w * s.w, b.w * c.w + b.z * s.w};
        }
    } else {
        for (int i = j; i < half && i < j + 4; i++) {
            const int e = r.halves ? i : 2 * i, f = r.halves ? half + i : 2 * i + 1;
            const float a = x[e], b = x[f], c = cs[i], s = cs[kMaxPairs + i];
            y[e] = a * c - b * s;
            y[f] = b * c + a * s;
        }
    }
}

template <int kType>
__device__ __forceinline__ uint16_t rounded(float v) {
    if constexpr (kType == kKvF16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// A token's scale in an int8 cache: absmax / 127 over its head's channels, which `lanes` neighbouring lanes hold (the channels past dim
// are zeros). `top`: the largest bits of the lane's magnitudes, which are ordered like them, NaN above all. A scale too small for its
// reciprocal (a head below 4e-37) is taken as zero.
struct Scaled {
    float scale, inv;
};
__device__ __forceinline__ Scaled token_scale(uint32_t top, int lanes) {
    for (int off = lanes / 2; off >= 1; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
    const float scale = as_float(top) / 127.0f, inv = 1.0f / scale;
    if (scale >= 0.0f && !(inv < __builtin_inff())) return Scaled{0.0f, 0.0f};
    return Scaled{scale, inv};
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, fabsf(v)); }
__device__ __forceinline__ uint32_t quant(float v, float inv) {
    return (uint32_t)((int)fminf(fmaxf(rintf(v * inv), -127.0f), 127.0f) + 128) & 0xffu;
}

// Eight channels of a token's keys into its block.
template <int kType>
__device__ __forceinline__ void store_key(const KvPool& p, char* block, int t, int d, const float (&o)[8], bool live) {
    if constexpr (kType == kKvI8) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, magnitude(o[i]));
        const Scaled s = token_scale(top, p.dp / 8);
        if (!live) return;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) w[i >> 2] |= quant(o[i], s.inv) << (8 * (i & 3));
        *(u32x2*)(block + kv_key_at(true, p.dp, t, d)) = u32x2{w[0], w[1]};
        if (d == 0) ((float*)(block + 2 * kv_plane_bytes(kType, p.dp)))[t] = s.scale;
    } else {
        if (!live) return;
        uint16_t h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = rounded<kType>(o[i]);
        *(u32x4*)(block + kv_key_at(false, p.dp, t, d)) =
            u32x4{(uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16, (uint32_t)h[4] | (uint32_t)h[5] << 16,
                  (uint32_t)h[6] | (uint32_t)h[7] << 16};
    }
}

// The new tokens' values of one block of the cache (at most rows / 32 + 2 a request), a share of its heads: a thread has four channels
// of the eight tokens that lie together in it, and writes them as one piece each. (Token by token, in the rows' workgroups, a store had
// a lane's 2 bytes in every 16: 4096 rows 54.6 us, 1297 rows 17.6.) by_rows: item is a row, and has its block if no row before it has.
template <int kType>
__device__ __forceinline__ void append_values(const KvAppendArgs& a, int item, int part, bool by_rows) {
    const KvPool& p = a.pool;
    const KvBatch& b = a.batch;
    int r = 0, before = 0;
    if (by_rows) {
        const KvRowPlace at = kv_row_place(b, item, b.rows);
        if (at.r < 0 || at.place < 0 || (at.place % kKvBlock && !at.first)) return;
        r = at.r;
        item = at.place / kKvBlock;
    } else {
        const bool any = kv_find(b.requests, item, r, before, [&](int q) {
            const int n = kv_rows(b, q).n, len = kv_length(b, q), from = max(len - n, 0);
            return n && len > from ? ((len - 1) / kKvBlock) - from / kKvBlock + 1 : 0;
        });
        if (!any) return;
        item += max(kv_length(b, r) - kv_rows(b, r).n, 0) / kKvBlock;
    }
    const KvRows m = kv_rows(b, r);
    const int len = kv_length(b, r), start = len - m.n;  // the first row's token, before the first if negative
    const int block = item, entry = block / (p.page / kKvBlock);
    if (entry >= b.width) return;
    const int page = b.tables[(size_t)r * b.width + entry];
    if (page < 0 || page >= p.pages) return;
    const int quads = p.dp >> 2, u = part * 256 + (int)threadIdx.x, quad = u % quads, g = (u / quads) & 3, head = u / (4 * quads);
    if (head >= p.kv_heads) return;
    const int d = 4 * quad;
    const bool live = d < p.dim;
    float x[8][4];
    uint32_t here = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int token = block * kKvBlock + (i >> 2) * 16 + g * 4 + (i & 3), row = token - start;
        f32x4u v = {0, 0, 0, 0};
        if (token < len && row >= 0) {
            here |= 1u << i;
            if (live) v = *(const f32x4u*)(a.v + ((size_t)(m.first + row) * p.kv_heads + head) * p.dim + d);
        }
#pragma unroll
        for (int c = 0; c < 4; c++) x[i][c] = v[c];
    }
    char* at = kv_block(p, page, head, block & (p.page / kKvBlock - 1));
    char* plane = at + kv_plane_bytes(kType, p.dp);
    if constexpr (kType == kKvI8) {
        float inv[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < 4; c++) top = max(top, magnitude(x[i][c]));
            const Scaled s = token_scale(top, quads);
            inv[i] = s.inv;
            if (quad == 0 && (here >> i & 1))
                ((float*)(at + 2 * kv_plane_bytes(kType, p.dp)))[kKvBlock + (i >> 2) * 16 + g * 4 + (i & 3)] = s.scale;
        }
        if (!live) return;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            char* to = plane + kv_value_at(true, 4 * g, d + c);
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) w[i >> 2] |= quant(x[i][c], inv[i]) << (8 * (i & 3));
            if (here == 0xff) {
                *(u32x2*)to = u32x2{w[0], w[1]};
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (here >> i & 1) to[i] = (char)(w[i >> 2] >> (8 * (i & 3)));
            }
        }
    } else {
        if (!live) return;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            char* to = plane + kv_value_at(false, 4 * g, d + c);
            uint16_t h[8];
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = rounded<kType>(x[i][c]);
            if (here == 0xff) {
                *(u32x4*)to = u32x4{(uint32_t)h[0] | (uint32_t)h[1] << 16, (uint32_t)h[2] | (uint32_t)h[3] << 16,
                                    (uint32_t)h[4] | (uint32_t)h[5] << 16, (uint32_t)h[6] | (uint32_t)h[7] << 16};
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (here >> i & 1) ((uint16_t*)to)[i] = h[i];
            }
        }
    }
}

template <int kType, bool kFast>
__global__ __launch_bounds__(256) void kv_append_kernel(KvAppendArgs a, int parts, int value_blocks, int value_parts, bool by_rows) {
    __shared__ float cs[2 * kMaxPairs];
    int index = blockIdx.x;
    if (index < value_blocks * value_parts) {
        append_values<kType>(a, index / value_parts, index % value_parts, by_rows);
        return;
    }
    index -= value_blocks * value_parts;
    // 32 consecutive rows go to one XCD (workgroups are dealt round the eight in turn): they share the lines of the keys' blocks.
    const int part = parts == 1 ? 0 : index % parts;
    const int row = parts == 1 ? (index >> 8) * 256 + (index & 7) * 32 + ((index >> 3) & 31) : index / parts;
    if (row >= a.batch.rows) return;
    const int tid = threadIdx.x;
    const KvRowPlace at = kv_row_place(a.batch, row, a.batch.rows);
    if (at.r < 0) return;
    const int r = at.r, place = at.place;
    const KvRope& rope = a.rope;
    for (int j = tid; j < rope.rotary >> 1; j += 256) {
        int position = place;
        if (rope.positions) {
            const int axis = rope.axes ? rope.axes[j] : 0;
            position = axis >= 0 && axis < rope.n_axes ? rope.positions[(size_t)axis * a.batch.rows + row] : 0;
        }
        const Turn t = turn_of(position, rope.freq[j], rope.scale);
        cs[j] = t.c;
        cs[kMaxPairs + j] = t.s;
    }
    __syncthreads();
    const int step = 256 * parts, from = part * 256 + tid, dim = a.pool.dim;
    if (a.q) {
        const int units = (((rope.rotary >> 1) + 3) >> 2) + ((dim - rope.rotary + 3) >> 2);
        const float* x = a.q + (size_t)row * a.heads * dim;
        float* y = a.q_out + (size_t)row * a.heads * dim;
        for (int u = from; u < a.heads * units; u += step) {
            const int h = u / units;
            rotate_query<kFast>(x + h * dim, y + h * dim, dim, u - h * units, rope, cs);
        }
    }
    if (!a.k || place < 0) return;
    const int in_page = place % a.pool.page, entry = place / a.pool.page;
    if (entry >= a.batch.width) return;
    const int page = a.batch.tables[(size_t)r * a.batch.width + entry];
    if (page < 0 || page >= a.pool.pages) return;
    // a head's channels in neighbouring lanes; whole head groups of lanes run together
    const int units = a.pool.dp >> 3;
    for (int u = from; u < a.pool.kv_heads * units; u += step) {
        const int h = u / units, d = (u - h * units) * 8;
        char* block = kv_block(a.pool, page, h, in_page / kKvBlock);
        float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const bool live = d < dim;
        if (live) rotated8<kFast>(a.k + ((size_t)row * a.pool.kv_heads + h) * dim, d, rope, cs, o);
        store_key<kType>(a.pool, block, in_page % kKvBlock, d, o, live);
    }
}

// What a stored key's eight channels stand for.
template <int kType>
__device__ __forceinline__ void load8(const KvPool& p, const char* block, int t, int d, float (&o)[8]) {
    const char* at = block + kv_key_at(kType == kKvI8, p.dp, t, d);
    if constexpr (kType == kKvI8) {
        const float scale = ((const float*)(block + 2 * kv_plane_bytes(kType, p.dp)))[t];
        const u32x2 w = *(const u32x2*)at;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = (float)((int)((w[i >> 2] >> (8 * (i & 3))) & 0xff) - 128) * scale;
    } else {
        const u32x4 w = *(const u32x4*)at;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint16_t h = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
            o[i] = kType == kKvF16 ? (float)__builtin_bit_cast(_Float16, h) : as_float((uint32_t)h << 16);
        }
    }
}

// The sum of the keys of each page that a call has filled: in fp64 in the order of the tokens, rounded to fp32 once. A workgroup per
// page that ends among the new tokens (at most rows / page + 1 a request; by_rows: a workgroup per row) and key head.
template <int kType>
__global__ __launch_bounds__(256) void kv_sums_kernel(KvPool p, KvBatch b, bool by_rows) {
    __shared__ double part[256 * 8];
    int item = blockIdx.x, r = 0, before = 0;
    if (by_rows) {
        const KvRowPlace at = kv_row_place(b, item, b.rows);
        if (at.r < 0 || at.place < 0 || (at.place + 1) % p.page) return;
        r = at.r;
        item = at.place / p.page;
    } else {
        const bool any = kv_find(b.requests, item, r, before, [&](int q) {
            const int n = kv_rows(b, q).n, len = kv_length(b, q);
            const int from = len - n > 0 ? len - n : 0;
            return n && len > from ? len / p.page - from / p.page : 0;
        });
        if (!any) return;
        item += max(kv_length(b, r) - kv_rows(b, r).n, 0) / p.page;
    }
    const int entry = item;
    if (entry >= b.width) return;
    const int page = b.tables[(size_t)r * b.width + entry];
    if (page < 0 || page >= p.pages) return;
    const int h = blockIdx.y, units = p.dp >> 3, groups = 256 / units, tid = threadIdx.x;
    const int u = tid % units, g = tid / units;
    double s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (g < groups) {
        for (int t = g; t < p.page; t += groups) {
            float o[8];
            load8<kType>(p, kv_block(p, page, h, t / kKvBlock), t % kKvBlock, 8 * u, o);
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] += (double)o[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) part[(g * units + u) * 8 + i] = s[i];
    }
    __syncthreads();
    for (int d = tid; d < p.dim; d += 256) {
        double sum = 0;
        for (int i = 0; i < groups; i++) sum += part[i * units * 8 + d];
        p.sums[((size_t)page * p.kv_heads + h) * p.dim + d] = (float)sum;
    }
}

__global__ __launch_bounds__(256) void kv_clear_kernel(u32x4* p, size_t n) {
    const u32x4 zero = {0, 0, 0, 0};
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = zero;
}

}  // namespace

hipError_t launch_kv_clear(void* p, size_t bytes, hipStream_t st) {
    const size_t n = bytes / 16;
    kv_clear_kernel<<<(unsigned)(n < 2048 * 256 ? (n + 255) / 256 : 2048), 256, 0, st>>>((u32x4*)p, n);
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t st) {
    const int rot = a.rope.rotary, dim = a.pool.dim;
    const bool fast = rot % 16 == 0 && dim % 8 == 0;
    const int rows = a.batch.rows, requests = a.batch.requests < rows ? a.batch.requests : rows, parts = rows < 256 ? 4 : 1;
    // blocks that the new tokens lie in: of n tokens at most n, and at most (n + 62) / 32
    const int64_t blocks = ((int64_t)rows + 62 * (int64_t)requests) / 32;
    // One or two rows a request: a row is found by search, a block or a page by a walk over the requests (4096 requests of one row 80 us by
    // rows and 180 by blocks, with sums 97 and 870; of four, 1024 requests 78 and 61, 201 and 132).
    const bool by_rows = rows <= 2 * requests;
    const int value_blocks = !a.k ? 0 : (int)(blocks < rows && !by_rows ? blocks : rows);
    const int value_parts = (a.pool.kv_heads * a.pool.dp + 255) / 256;
    const unsigned grid = (unsigned)(value_blocks * value_parts + (parts == 1 ? (rows + 255) / 256 * 256 : rows * parts));
    auto go = [&](auto type, auto quick) {
        kv_append_kernel<decltype(type)::value, decltype(quick)::value><<<grid, 256, 0, st>>>(a, parts, value_blocks, value_parts, by_rows);
    };
    using std::integral_constant;
    auto typed = [&](auto type) {
        if (fast)
            go(type, std::true_type{});
        else
            go(type, std::false_type{});
    };
    switch (a.pool.type) {
        case kKvF16: typed(integral_constant<int, kKvF16>{}); break;
        case kKvBf16: typed(integral_constant<int, kKvBf16>{}); break;
        default: typed(integral_constant<int, kKvI8>{});
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.pool.sums || !a.k) return e;
    const int64_t ends = by_rows ? rows : (int64_t)rows / a.pool.page + requests;
    const dim3 pages((unsigned)ends, (unsigned)a.pool.kv_heads);
    switch (a.pool.type) {
        case kKvF16: kv_sums_kernel<kKvF16><<<pages, 256, 0, st>>>(a.pool, a.batch, by_rows); break;
        case kKvBf16: kv_sums_kernel<kKvBf16><<<pages, 256, 0, st>>>(a.pool, a.batch, by_rows); break;
        default: kv_sums_kernel<kKvI8><<<pages, 256, 0, st>>>(a.pool, a.batch, by_rows);
    }
    return hipGetLastError();
}

}  // namespace ovfq
