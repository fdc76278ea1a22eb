// attend_few.hip — attention of few columns (up to 32 (row, query head) pairs of a request and key head: decode steps, drafted tokens)
// over a paged cache, of any columns over selected pages, and the joining of partial outputs. Arithmetic: attend.h.
//
// Bound: HBM, each key and value is read once for its request. Four waves take a piece's blocks in turn, each through a ring of its own
// in LDS that the DMA fills in operand order (no transposition, no barriers): a block's keys are loaded while the block before it goes
// through its softmax and second product, its values during its own first one. Keys and values loaded into registers instead, with as
// many under way, are 1 to 2 % faster on one column tile (64 decode rows of 5 k tokens 237 / 239 us), but two tiles leave a wave a SIMD
// then (60 drafted rows, 8-bit cache, 150 / 112). Pieces are cut so that all key heads together give a few workgroups for each CU
// whatever the lengths; their partial outputs are joined by a second launch (by the tile's last
// workgroup, over agent-scope stores and a counter, it took as long: one row 12.0 us and 12.6, 60 drafted rows 101 and 95). Waves join
// theirs in LDS, in a fixed order.
#include <type_traits>

#include "attend.h"

namespace ovfq {

namespace {

// Blocks that a wave has under way: rings of half of a CU's LDS at most (all of it for heads past 128), so that two workgroups fit.
constexpr int few_depth(int type, int dp) { return dp > 128 ? 1 : 18432 / kv_bytes(type, dp); }

template <int kType, int kDp, int kCols, bool kSelected>
__global__ __launch_bounds__(256, kDp <= 128 ? 2 : 1) void attend_few_kernel(AttendArgs a, Cut cut) {
    using Att = Attention<kType, kDp, kCols>;
    using M = KvMath<kType>;
    constexpr int kPlane = kv_plane_bytes(kType, kDp), kBytes = kv_bytes(kType, kDp), kLoads = kPlane / 1024;
    constexpr int kKeyLoads = kLoads + (kType == kKvI8 ? 1 : 0), kLoadsOfBlock = kKeyLoads + kLoads;
    constexpr int kDepth = few_depth(kType, kDp);
    __shared__ __attribute__((aligned(16))) char shared[4 * kDepth * kBytes];  // the waves' rings, then the join of their outputs
    f32x4(*joined)[kCols * Att::kTiles][64] = (f32x4(*)[kCols * Att::kTiles][64])shared;
    static_assert(2 * kCols * Att::kTiles * 64 * 16 <= 4 * kDepth * kBytes, "the join fits into the rings");
    __shared__ float refs[4][kCols * 16];
    __shared__ float sums[4][kCols * 16];
    const KvPool& pool = a.pool;
    const KvBatch& b = a.batch;
    const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 15;
    const int head = (int)(blockIdx.x % (unsigned)pool.kv_heads), item = (int)(blockIdx.x / (unsigned)pool.kv_heads);
    TileWork w;
    int whole = 0;  // selected: the row's pages, and how many
    const int* pages = nullptr;
    const int shift = 31 - __builtin_clz(pool.page / kKvBlock);
    if constexpr (kSelected) {
        // item: row, tile of query heads, piece
        const int tiles = (cut.group + 15) >> 4, per = tiles * cut.target;
        const int row = item / per;
        const int r = a.where[row];
        if (r < 0) return;
        const KvRows m = kv_rows(b, r);
        w.r = r;
        w.first_row = row;
        w.rows = 1;
        w.place = kv_length(b, r) - m.n + (row - m.first);
        w.tile = (item - row * per) / cut.target;
        w.piece = (item - row * per) % cut.target;
        w.col0 = 16 * w.tile;
        w.slot = item - w.piece;
        w.tile_index = item / cut.target;
        pages = a.chosen + ((size_t)row * pool.kv_heads + head) * a.top;
        for (int i = 0; i < a.top; i += 64) whole += __popcll(__ballot(i + lane < a.top && pages[min(i + lane, a.top - 1)] >= 0));
        const int blocks = whole << shift, each = cut.least_blocks;
        w.pieces = blocks > each ? (blocks + each - 1) / each : 1;
        if (w.piece >= w.pieces) return;
        w.block0 = w.piece * each;
        w.block1 = min(blocks, w.block0 + each);
    } else {
        if (!cut_item(cut, pool, b, a.plan, item, w)) return;
    }
    if (a.plans && threadIdx.x == 0 && w.piece == 0 && head == 0) a.plans[w.tile_index] = w;
    Att att;
#pragma unroll
    for (int t = 0; t < kCols; t++) {
        const int c = w.col0 + 16 * t + col, i = c / cut.group;
        const int qh = head * cut.group + (c - i * cut.group), last = w.place + i;
        typename Att::Row row;
        Att::fetch(row, a.q + ((size_t)(w.first_row + i) * a.heads + qh) * pool.dim, i < w.rows, pool.dim);
        att.column(t, i < w.rows, first_seen(last, a.window), last);
        att.query(t, row, i < w.rows, pool.dim, a.scale * kLog2e);
    }
    const int first_last = w.place + w.col0 / cut.group;  // the tile's rows see up to first_last .. last_last
    const int last_last = w.place + min(w.rows - 1, (w.col0 + 16 * kCols - 1) / cut.group);
    const int last_low = first_seen(last_last, a.window);

    const int* table = b.tables + (size_t)w.r * b.width;
    BlockWalk walk;
    int held = 0, phys = -1;  // selected: lanes' page numbers in the request's table, and in the cache
    auto block_of = [&](int i) { return w.block0 + wave + 4 * i; };
    const int mine = w.block1 > w.block0 + wave ? (w.block1 - w.block0 - wave + 3) >> 2 : 0;
    auto selected_fetch = [&](int i) {
        const int at = (block_of(i) + 4 * lane) >> shift;
        const int p = at < whole ? pages[at] : -1;
        held = p;
        const int t = p >= 0 && p < b.width ? table[p] : -1;
        phys = t >= 0 && t < pool.pages ? t : -1;
    };
    // a block's page (-1: not there, its tokens count as hidden), first token and bytes, in rising order
    struct At {
        int page, first;
        const char* bytes;
    };
    auto locate = [&](int i) {
        At at;
        const int block = block_of(i), within = block & ((1 << shift) - 1);
        if constexpr (kSelected) {
            if (i && (i & 63) == 0) selected_fetch(i);
            at.page = __builtin_amdgcn_readlane(phys, i & 63);
            at.first = __builtin_amdgcn_readlane(held, i & 63) * pool.page + within * kKvBlock;
        } else {
            at.page = walk.page(i);
            at.first = block * kKvBlock;
        }
        at.bytes = kv_block(pool, max(at.page, 0), head, within);
        return at;
    };
    auto stage = [&](char* dst, const char* src, bool values) {
        const int plane = values ? kPlane : 0;
#pragma unroll
        for (int k = 0; k < kLoads; k++)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + plane + k * 1024 + lane * 16),
                                             (__attribute__((address_space(3))) void*)(dst + plane + k * 1024), 16, 0, 0);
        if constexpr (kType == kKvI8) {
            if (!values)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + 2 * kPlane + lane * 4),
                                                 (__attribute__((address_space(3))) void*)(dst + 2 * kPlane), 4, 0, 0);
        }
    };
    if (mine) {
        if constexpr (kSelected)
            selected_fetch(0);
        else
            walk.start(pool, table, b.width, block_of(0), 4);
        char* ring = shared + wave * kDepth * kBytes;
        At ahead[kDepth];  // blocks i .. i + kDepth - 1
#pragma unroll
        for (int j = 0; j < kDepth; j++) {
            ahead[j] = j && j >= mine ? ahead[j ? j - 1 : 0] : locate(j);
            stage(ring + j * kBytes, ahead[j].bytes, false);
            stage(ring + j * kBytes, ahead[j].bytes, true);
        }
        int slot = 0;
        for (int i = 0; i < mine; i++) {
            const At now = ahead[0];
            // (past the last block its predecessor is loaded again: the counts of loads under way stay)
            const At next = i + kDepth < mine ? locate(i + kDepth) : ahead[kDepth - 1];
            char* place = ring + slot * kBytes;
            const char* at = place + lane * 16;
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads + (kDepth - 1) * kLoadsOfBlock) : "memory");
            f32x4 ks[2] = {}, vs[2] = {};
            if constexpr (kType == kKvI8) {
                const char* c = place + 2 * kPlane + (lane >> 4) * 16;
                ks[0] = *(const f32x4*)c;
                ks[1] = *(const f32x4*)(c + 64);
                vs[0] = *(const f32x4*)(c + 128);
                vs[1] = *(const f32x4*)(c + 192);
            }
            f32x4 s[kCols][2];
            att.scores(s, [&](int tile, int chunk) {
                return key_operand<kType, kDp>(tile, chunk, [&](int off) { return *(const u32x4*)(at + off); });
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the keys are read: their place takes the next ones
            stage(place, next.bytes, false);
            const bool masked = now.first + kKvBlock - 1 > first_last || now.first < last_low;
            u32x4 p[kCols][M::kParts];
            if (now.page >= 0) {
                att.settle(s, masked, now.first, ks);
                att.probabilities(s, p, masked, now.first, vs);
            }
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kKeyLoads + (kDepth - 1) * kLoadsOfBlock) : "memory");
            if (now.page >= 0) {
                auto value = [&](int tile) {
                    return value_operand<kType, kDp>(tile, [&](int off) { return *(const u32x4*)(at + off); });
                };
                if constexpr (kType != kKvI8) {
                    if (masked) {
                        bool any = false;
                        for (int k = 0; k < kLoads; k++) any = any | any_not_finite<kType>(*(const u32x4*)(at + kPlane + k * 1024));
                        if (__ballot(any)) {
                            att.note_bad(now.first, value);
                            for (int k = 0; k < kLoads; k++) {
                                u32x4* v = (u32x4*)(place + kPlane + k * 1024 + lane * 16);
                                *v = finite_part<kType>(*v);
                            }
                        }
                    }
                }
                att.products(p, value);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            stage(place, next.bytes, true);
            slot = slot + 1 < kDepth ? slot + 1 : 0;
#pragma unroll
            for (int j = 0; j + 1 < kDepth; j++) ahead[j] = ahead[j + 1];
            ahead[kDepth - 1] = next;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last loads land before their places serve the join
    }
    __syncthreads();
    att.close();
    // join the waves: 2 and 3 into 0 and 1, then 1 into 0
    if (lane < 16) {
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            refs[wave][16 * t + lane] = att.ref[t];
            sums[wave][16 * t + lane] = att.l[t];
        }
    }
    __syncthreads();
    float top[kCols], l[kCols];
#pragma unroll
    for (int t = 0; t < kCols; t++) {
        const int c = 16 * t + col;
        top[t] = fmaxf(fmaxf(refs[0][c], refs[1][c]), fmaxf(refs[2][c], refs[3][c]));
        const float m = top[t] == -kInf ? 0.0f : top[t];
        l[t] = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; v++) l[t] += sums[v][c] * __builtin_amdgcn_exp2f(refs[v][c] - m);
        const float f = __builtin_amdgcn_exp2f(att.ref[t] - m) * one_over(l[t]);
#pragma unroll
        for (int d = 0; d < Att::kTiles; d++) att.o[t][d] = att.output(t, d, f);
    }
    for (int from = 2; from >= 1; from >>= 1) {
        if (wave >= from && wave < 2 * from) {
#pragma unroll
            for (int t = 0; t < kCols; t++)
#pragma unroll
                for (int d = 0; d < Att::kTiles; d++) joined[wave - from][t * Att::kTiles + d][lane] = att.o[t][d];
        }
        __syncthreads();
        if (wave < from) {
#pragma unroll
            for (int t = 0; t < kCols; t++)
#pragma unroll
                for (int d = 0; d < Att::kTiles; d++) att.o[t][d] += joined[wave][t * Att::kTiles + d][lane];
        }
        __syncthreads();
    }
    if (wave) return;
    if (w.pieces > 1) {
        float* part = a.parts + ((size_t)(w.slot + w.piece) * pool.kv_heads + head) * (size_t)part_floats(16 * kCols, kDp);
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            if (lane < 16) {
                part[32 * t + lane] = top[t];
                part[32 * t + 16 + lane] = l[t];
            }
#pragma unroll
            for (int d = 0; d < Att::kTiles; d++)
                *(f32x4*)(part + 32 * kCols + ((t * Att::kTiles + d) * 64 + lane) * 4) = att.o[t][d];
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < kCols; t++) {
        const int c = w.col0 + 16 * t + col, i = c / cut.group;
        if (i >= w.rows) continue;
        float* y = a.out + ((size_t)(w.first_row + i) * a.heads + head * cut.group + (c - i * cut.group)) * pool.dim;
#pragma unroll
        for (int d = 0; d < Att::kTiles; d++) {
            const int at = 16 * d + 4 * (lane >> 4);
            if (at < pool.dim) *(f32x4u*)(y + at) = att.o[t][d];
        }
    }
}

}  // namespace

// Joins the pieces of each tile: out = sum w o / sum w with w = 2^(ref - top) l, in a fixed order. A workgroup per 16 columns of a tile,
// key head and 16 channels * `wide` (blockIdx.y; blockIdx.z: the tiles past what x takes): a thread has a column that is used and four
// channels, and what is left of the workgroup's threads shares the pieces.
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a, Cut cut, int dp, int wide) {
    __shared__ float tops[16][16], ls[16][16];
    __shared__ f32x4 part_o[256];
    const KvPool& pool = a.pool;
    const int subs = 1 << (cut.cols_log2 - 4), cols = 16 * subs, tid = threadIdx.x;
    const int head = (int)(blockIdx.x % (unsigned)pool.kv_heads);
    const int item = (int)((blockIdx.x + blockIdx.z * gridDim.x) / (unsigned)pool.kv_heads), index = item / subs, sub = item - index * subs;
    const int head_tiles = (cut.group + 15) >> 4;
    const TilePlan w = a.plans[min(index, cut.tiles - 1)];  // (under way beside the count)
    if (index >= (a.where ? a.batch.rows * head_tiles : a.plan->joins)) return;
    if (a.where && a.where[index / head_tiles] < 0) return;
    // (a plan that nothing wrote, for offsets that overlap, must not lead out of the planes)
    if (w.pieces <= 1 || w.slot < 0 || w.slot > cut.slots - w.pieces || w.first_row < 0 || w.rows <= 0 ||
        w.rows > a.batch.rows - w.first_row || w.col0 < 0 || w.col0 >= w.rows * cut.group)
        return;
    const int first = w.col0 + 16 * sub, used = min(16, w.rows * cut.group - first);
    if (used <= 0) return;
    const size_t stride = (size_t)part_floats(cols, dp) * pool.kv_heads;
    const float* base = a.parts + ((size_t)w.slot * pool.kv_heads + head) * (size_t)part_floats(cols, dp);
    const float* ml = base + 32 * sub;
    {  // the columns' tops and sums: 16 threads a column
        const int col = tid & 15, share = tid >> 4;
        float top = -kInf;
        for (int j = share; j < w.pieces; j += 16) top = fmaxf(top, ml[j * stride + col]);
        tops[share][col] = top;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; k++) top = fmaxf(top, tops[k][col]);
        const float m = top == -kInf ? 0.0f : top;
        float l = 0.0f;
        for (int j = share; j < w.pieces; j += 16) l += ml[j * stride + 16 + col] * __builtin_amdgcn_exp2f(ml[j * stride + col] - m);
        ls[share][col] = l;
        __syncthreads();
        if (share == 0) {
            tops[0][col] = m;
            l = 0.0f;
#pragma unroll
            for (int k = 0; k < 16; k++) l += ls[k][col];
            ls[0][col] = one_over(l);
        }
        __syncthreads();
    }
    const int tiles = dp >> 4, d0 = (int)blockIdx.y * wide, quads = min(wide, tiles - d0) * 4;
    const int units = used * quads, shares = units >= 256 ? 1 : 256 / units;
    for (int u0 = 0; u0 < units; u0 += 256) {
        const int share = shares == 1 ? 0 : tid / units, u = shares == 1 ? u0 + tid : tid - share * units;
        const bool live = u < units && share < shares;
        const int col = live ? u % used : 0, quad = live ? u / used : 0, d = d0 + (quad >> 2), g = quad & 3;
        f32x4 o = {0, 0, 0, 0};
        if (live) {
            const float m = tops[0][col], inv = ls[0][col];
            const float* mine = base + 32 * subs + ((sub * tiles + d) * 64 + g * 16 + col) * 4;
#pragma unroll 4
            for (int j = share; j < w.pieces; j += shares) {
                const float f = ml[j * stride + 16 + col] * __builtin_amdgcn_exp2f(ml[j * stride + col] - m) * inv;
                o += *(const f32x4*)(mine + j * stride) * f;
            }
        }
        if (shares > 1) {
            part_o[tid] = o;
            __syncthreads();
            if (share == 0)
                for (int k = 1; k < shares; k++) o += part_o[tid + k * units];
        }
        if (!live || share) continue;
        const int c = first + col, i = c / cut.group, at = 16 * d + 4 * g;
        if (at < pool.dim)
            *(f32x4u*)(a.out + ((size_t)(w.first_row + i) * a.heads + head * cut.group + (c - i * cut.group)) * pool.dim + at) = o;
    }
}

hipError_t launch_attend_few(const AttendArgs& a, const Cut& cut, unsigned items, hipStream_t st) {
    const unsigned grid = items * (unsigned)a.pool.kv_heads;
    auto go = [&](auto type, auto dp) {
        constexpr int kType = decltype(type)::value, kDp = decltype(dp)::value;
        if constexpr (kType != kKvI8 || kDp != 96) {
            if (a.where)
                attend_few_kernel<kType, kDp, 1, true><<<grid, 256, 0, st>>>(a, cut);
            else if (cut.cols_log2 == 4)
                attend_few_kernel<kType, kDp, 1, false><<<grid, 256, 0, st>>>(a, cut);
            else if constexpr (kDp <= 128)
                attend_few_kernel<kType, kDp, 2, false><<<grid, 256, 0, st>>>(a, cut);
        }
    };
    using std::integral_constant;
    auto sized = [&](auto type) {
        switch (a.pool.dp) {
            case 64: go(type, integral_constant<int, 64>{}); break;
            case 96: go(type, integral_constant<int, 96>{}); break;
            case 128: go(type, integral_constant<int, 128>{}); break;
            default: go(type, integral_constant<int, 256>{});
        }
    };
    switch (a.pool.type) {
        case kKvF16: sized(integral_constant<int, kKvF16>{}); break;
        case kKvBf16: sized(integral_constant<int, kKvBf16>{}); break;
        default: sized(integral_constant<int, kKvI8>{});
    }
    return hipGetLastError();
}

hipError_t launch_attend_join(const AttendArgs& a, const Cut& cut, unsigned tiles, hipStream_t st) {
    const unsigned heads = (unsigned)a.pool.kv_heads, most = (1u << 20) / heads, subs = tiles << (cut.cols_log2 - 4);
    const unsigned x = (subs < most ? subs : most) * heads, z = (subs + most - 1) / most, all = (unsigned)a.pool.dp >> 4;
    const unsigned wide = x >= 512 ? all : x >= 128 ? 2 : 1;  // few tiles: their channels over several workgroups
    attend_join_kernel<<<dim3(x, (all + wide - 1) / wide, z), 256, 0, st>>>(a, cut, a.pool.dp, (int)wide);
    return hipGetLastError();
}

}  // namespace ovfq
