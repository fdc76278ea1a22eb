// attend_many.hip — attention of many columns (prompts, chunks of them) over a paged cache. Arithmetic: attend.h.
//
// Bound: MFMA, 4 D flops per (column, token) times the parts that q and p are split in (two fp16, three bf16), beside the softmax's
// vector work. Four waves of 16 kCols columns each share a tile; a block's keys and values go to LDS once for all of them, by DMA in
// the operand order that they have in memory (reads of it are 1 KiB in a row, free of conflicts), one block ahead. Workgroups of one
// key head come to one XCD where the head count allows, so its blocks are read from HBM once.
#include <type_traits>

#include "attend.h"

namespace ovfq {

namespace {

template <int kType, int kDp, int kCols>
__global__ __launch_bounds__(256, 2) void attend_many_kernel(AttendArgs a, Cut cut) {
    using Att = Attention<kType, kDp, kCols>;
    using M = KvMath<kType>;
    constexpr int kBytes = kv_bytes(kType, kDp), kPlane = kv_plane_bytes(kType, kDp);
    __shared__ __attribute__((aligned(16))) char ring[2][kBytes];
    const KvPool& pool = a.pool;
    const KvBatch& b = a.batch;
    const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 15;
    const int head = (int)(blockIdx.x % (unsigned)pool.kv_heads), item = (int)(blockIdx.x / (unsigned)pool.kv_heads);
    TileWork w;
    if (!(b.requests <= 64 ? cut_tiles(cut, pool, b, a.plan, item, w) : cut_item(cut, pool, b, a.plan, item, w))) return;
    if (a.plans && threadIdx.x == 0 && w.piece == 0 && head == 0) a.plans[w.tile_index] = w;
    const int wave_col = w.col0 + 16 * kCols * wave;
    BlockWalk walk;
    const int blocks = max(w.block1 - w.block0, 0);
    const int in_page = pool.page / kKvBlock - 1;
    walk.start(pool, b.tables + (size_t)w.r * b.width, b.width, w.block0, 1);
    auto stage = [&](int i, int page) {
        const char* src = kv_block(pool, page, head, (w.block0 + i) & in_page);
        char* dst = ring[i & 1];
        constexpr int kPieces = 2 * kPlane / 1024;
#pragma unroll
        for (int k = 0; k < kPieces; k += 4)
            if (kPieces % 4 == 0 || k + wave < kPieces)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + (k + wave) * 1024 + lane * 16),
                                                 (__attribute__((address_space(3))) void*)(dst + (k + wave) * 1024), 16, 0, 0);
        if constexpr (kType == kKvI8) {
            if (wave == 0)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + 2 * kPlane + lane * 4),
                                                 (__attribute__((address_space(3))) void*)(dst + 2 * kPlane), 4, 0, 0);
        }
    };
    typename Att::Row rows[kCols];  // (of columns that are not used the first row: at a branch's end the compiler would wait for the loads)
#pragma unroll
    for (int t = 0; t < kCols; t++) {
        const int c = wave_col + 16 * t + col, i = c / cut.group, qh = head * cut.group + (c - i * cut.group);
        Att::fetch(rows[t], a.q + ((size_t)(w.first_row + (i < w.rows ? i : 0)) * a.heads + qh) * pool.dim, true, pool.dim);
    }
    asm volatile("" ::: "memory");  // (the table's, the queries' and the first block's loads are on their way together)
    int page = blocks ? walk.page(0) : -1;
    stage(0, max(page, 0));
    asm volatile("" ::: "memory");
    Att att;
#pragma unroll
    for (int t = 0; t < kCols; t++) {
        const int i = (wave_col + 16 * t + col) / cut.group, last = w.place + i;
        att.column(t, i < w.rows, first_seen(last, a.window), last);
        att.query(t, rows[t], i < w.rows, pool.dim, a.scale * kLog2e);
    }
    // what the wave's rows see
    const int i0 = wave_col / cut.group, i1 = min(w.rows - 1, (wave_col + 16 * kCols - 1) / cut.group);
    const bool live = i0 < w.rows;
    const int first_last = w.place + i0, last_last = w.place + i1;
    const int first_low = first_seen(first_last, a.window), last_low = first_seen(last_last, a.window);
    // and the least that a column of the tile sees
    const int tile_last = w.place + w.col0 / cut.group;
    const int tile_low = first_seen(w.place + min(w.rows - 1, (w.col0 + 64 * kCols - 1) / cut.group), a.window);

    for (int i = 0; i < blocks; i++) {
        const int next = i + 1 < blocks ? walk.page(i + 1) : -1;
        // this wave's share of block i has landed; behind the barrier all of it, and every wave is past the block before
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (next >= 0) stage(i + 1, next);
        const int first = (w.block0 + i) * kKvBlock;
        if constexpr (kType != kKvI8) {
            if (page >= 0 && (first + kKvBlock - 1 > tile_last || first < tile_low)) {  // masked for one of the tile's columns
                char* values = ring[i & 1] + kPlane;
                bool any = false;
                for (int k = threadIdx.x * 16; k < kPlane; k += 4096) any = any | any_not_finite<kType>(*(const u32x4*)(values + k));
                if (__syncthreads_or(any)) {
                    att.note_bad(first, [&](int tile) { return *(const u32x4*)(values + tile * 1024 + lane * 16); });
                    __syncthreads();
                    for (int k = threadIdx.x * 16; k < kPlane; k += 4096) *(u32x4*)(values + k) = finite_part<kType>(*(const u32x4*)(values + k));
                    __syncthreads();
                }
            }
        }
        if (page >= 0 && live && first <= last_last && first + (kKvBlock - 1) >= first_low) {
            const char* at = ring[i & 1] + lane * 16;
            f32x4 ks[2] = {}, vs[2] = {};
            if constexpr (kType == kKvI8) {
                const char* s = ring[i & 1] + 2 * kPlane + (lane >> 4) * 16;
                ks[0] = *(const f32x4*)s;
                ks[1] = *(const f32x4*)(s + 64);
                vs[0] = *(const f32x4*)(s + 128);
                vs[1] = *(const f32x4*)(s + 192);
            }
            auto load = [&](int off) { return *(const u32x4*)(at + off); };
            f32x4 s[kCols][2];
            att.scores(s, [&](int tile, int chunk) { return key_operand<kType, kDp>(tile, chunk, load); });
            const bool masked = first + kKvBlock - 1 > first_last || first < last_low;
            u32x4 p[kCols][M::kParts];
            att.settle(s, masked, first, ks);
            att.probabilities(s, p, masked, first, vs);
            att.products(p, [&](int tile) { return value_operand<kType, kDp>(tile, load); });
        }
        page = next;
    }
    if (!blocks) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the first one's load, which nothing waited for)
    att.close();
    if (w.pieces > 1) {
        float* part = a.parts + ((size_t)(w.slot + w.piece) * pool.kv_heads + head) * (size_t)part_floats(64 * kCols, kDp);
#pragma unroll
        for (int t = 0; t < kCols; t++) {
            const int sub = wave * kCols + t;
            const float inv = one_over(att.l[t]);
            if (lane < 16) {
                part[32 * sub + lane] = att.ref[t];
                part[32 * sub + 16 + lane] = att.l[t];
            }
#pragma unroll
            for (int d = 0; d < Att::kTiles; d++)
                *(f32x4*)(part + 32 * 4 * kCols + ((sub * Att::kTiles + d) * 64 + lane) * 4) = att.output(t, d, inv);
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < kCols; t++) {
        const int c = wave_col + 16 * t + col, i = c / cut.group;
        if (i >= w.rows) continue;
        const float inv = one_over(att.l[t]);
        float* y = a.out + ((size_t)(w.first_row + i) * a.heads + head * cut.group + (c - i * cut.group)) * pool.dim;
#pragma unroll
        for (int d = 0; d < Att::kTiles; d++) {
            const int at = 16 * d + 4 * (lane >> 4);
            if (at < pool.dim) *(f32x4u*)(y + at) = att.output(t, d, inv);
        }
    }
}

// Counts the items of each 64 requests, a wave each; every workgroup finds the pieces' size for itself.
__global__ __launch_bounds__(1024) void attend_plan_kernel(KvPool pool, KvBatch b, Cut c, CutPlan* plan) {
    __shared__ float sums[16];
    __shared__ int counts[16], spans[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    float sum = 0.0f;
    int tiles = 0, longest = 0;
    constexpr int kMostTiles = 1 << 24;  // more than a launch has room for: offsets that overlap may give any number, past 32 bits as well
    for (int r = tid; r < b.requests; r += 1024) {
        const CutRequest q = cut_load(c, pool, b, r);
        sum += q.sum;
        tiles = min(tiles + q.tiles, kMostTiles);
        longest = max(longest, q.blocks);
    }
    sum = wave_sum(sum);
    tiles = min(wave_sum(tiles), kMostTiles);
    longest = wave_max(longest);
    if (lane == 0) {
        sums[wave] = sum;
        counts[wave] = tiles;
        spans[wave] = longest;
    }
    __syncthreads();
    sum = 0.0f;
    tiles = longest = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        sum += sums[i];
        tiles += counts[i];
        longest = max(longest, spans[i]);
    }
    const float inv = 1.0f / cut_piece(c, sum, tiles);
    const bool fit = tiles <= c.tiles;  // (if not, offsets overlap: none of the call's tiles)
    if (blockIdx.x == 0 && tid == 0) *plan = CutPlan{fit && cut_pieces(longest, inv) > 1 ? tiles : 0, fit ? tiles : 0, inv, 0};
    const int chunk = (int)blockIdx.x * 16 + wave;
    if (64 * chunk >= b.requests) return;
    const CutRequest q = cut_load(c, pool, b, 64 * chunk + lane);
    const int2 mine = cut_items(q, inv);
    const CutChunk s{wave_sum(mine.x), wave_sum(q.tiles), wave_sum(mine.y), 0};
    if (lane == 0) ((CutChunk*)(plan + 1))[chunk] = s;
}

}  // namespace

hipError_t launch_attend_few(const AttendArgs& a, const Cut& cut, unsigned items, hipStream_t st);
hipError_t launch_attend_join(const AttendArgs& a, const Cut& cut, unsigned tiles, hipStream_t st);

namespace {

// Columns of a request that the few-column kernel takes.
int few_columns(const AttendArgs& a) { return a.pool.dp <= 128 ? 32 : 16; }

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

constexpr int kItems = 512;  // two workgroups a CU: registers and LDS
// More requests than that have their items counted by a launch of its own, whose 3 us are less than every workgroup's walk over them
// (single rows of 256 tokens: 65 requests 28.5 us with it and 25.9 without, 130 40.2 / 41.6, 300 73.9 / 93.1, 4096 835 / 4883).
constexpr int kPlanned = 128;

// A piece has at least so many blocks (8; with 4 and 16: one row over 1500 tokens 12.7 us, 12.2, 14.2; 64 rows over 2000 23.9, 24.3, 32.2; a
// prompt of 512 rows 26.2, 26.9, 29.7), and where there are tiles enough, one is cut if it is longer than so many times a workgroup's mean
// share: beside tiles of many columns 1.5 (with 1.0 and 2.5: a prompt of 2048 rows 95 us, 116, 105), of few 2 (with 1.5 and 3: 100 single
// rows over 100 to 16 k tokens 325, 332, 373).
constexpr int kLeastBlocks = 8;
constexpr float kSlackMany = 1.5f, kSlackFew = 2.0f;

struct Plan {
    Cut cut;
    bool split;
    unsigned items, tiles;  // most of a key head
};

// Which kernels a call takes: the few-column one where no request has more columns than it takes; else the other one, and the first
// beside it for the requests that it takes if the rows behind the longest request's are that few for each (a decode step with a chunk of a
// prompt in it: 512 rows over 8 k beside 31 single ones 344 us, all of them in the many-column kernel 457, where they waste three
// waves of four). A launch for nothing costs 6 to 8 us with its join, so prompts alone have one.
struct Kinds {
    bool few, many;
};
Kinds kinds_of(const AttendArgs& a) {
    const int64_t group = a.heads / a.pool.kv_heads, few = few_columns(a);
    if (a.batch.most * group <= few) return Kinds{true, false};
    return Kinds{a.batch.requests > 1 && group <= few && (a.batch.rows - a.batch.most) * group <= (a.batch.requests - 1) * few, true};
}

Plan plan_attend(const AttendArgs& a, bool few) {
    const Kinds kinds = kinds_of(a);
    const int group = a.heads / a.pool.kv_heads, requests = a.batch.requests < a.batch.rows ? a.batch.requests : a.batch.rows;
    Plan p{};
    p.split = true;
    int64_t most = (int64_t)a.batch.most * group;
    if (few && most > few_columns(a)) most = few_columns(a);
    // columns of a tile: 16 or 32, by the requests' most or, beside the other kernel, their mean
    const int64_t usual = kinds.many ? (int64_t)(a.batch.rows - a.batch.most) * group / (requests > 1 ? requests - 1 : 1) : most;
    const int log2 = few ? (usual <= 16 ? 4 : 5) : a.pool.dp <= 128 ? 7 : 6;
    const int least = !few && kinds.few ? few_columns(a) + 1 : 1;
    p.cut = Cut{log2, least, (int)most, ceil_div(kItems, a.pool.kv_heads), kLeastBlocks, few ? kSlackFew : kSlackMany, a.window, group, 0, 0, 0};
    p.tiles = (unsigned)(few ? requests * ceil_div(most, 1 << log2) : (((int64_t)a.batch.rows * group) >> log2) + requests);
    // Pieces are no longer than the mean by more than `slack`, and the sum of the tiles' lengths that it comes from is half of their number
    // times the longest at least: so many pieces at most, and so many of tiles that are cut.
    p.items = p.tiles + 2 * (unsigned)p.cut.target + 2;
    p.cut.slots = 4 * p.cut.target + 2;
    p.cut.tiles = (int)p.tiles;
    p.cut.planned = a.batch.requests > kPlanned;
    return p;
}

size_t rounded(size_t n) { return (n + 255) & ~size_t(255); }
size_t part_bytes(const AttendArgs& a, const Plan& p) {
    return rounded((size_t)p.cut.slots * a.pool.kv_heads * part_floats(1 << p.cut.cols_log2, a.pool.dp) * 4);
}
size_t cut_bytes(const AttendArgs& a, const Plan& p) {
    return rounded(sizeof(CutPlan) + (p.cut.planned ? (size_t)ceil_div(a.batch.requests, 64) * sizeof(CutChunk) : 0));
}
size_t plan_bytes(const AttendArgs& a, const Plan& p) { return cut_bytes(a, p) + rounded((size_t)p.tiles * sizeof(TilePlan)); }
AttendArgs with_scratch(const AttendArgs& a, const Plan& p) {
    AttendArgs m = a;
    if (p.split) {
        m.plan = (CutPlan*)((char*)a.parts + part_bytes(a, p));
        m.plans = (TilePlan*)((char*)m.plan + cut_bytes(a, p));
    }
    return m;
}
hipError_t launch_plan(const AttendArgs& a, const Plan& p, hipStream_t st) {
    if (!p.cut.planned) return hipSuccess;
    attend_plan_kernel<<<ceil_div(a.batch.requests, 1024), 1024, 0, st>>>(a.pool, a.batch, p.cut, a.plan);
    return hipGetLastError();
}

}  // namespace

size_t attend_scratch(const AttendArgs& a) {
    const Kinds kinds = kinds_of(a);
    const Plan few = plan_attend(a, true), many = plan_attend(a, false);
    return (kinds.few ? part_bytes(a, few) + plan_bytes(a, few) : 0) + (kinds.many ? part_bytes(a, many) + plan_bytes(a, many) : 0);
}

hipError_t launch_attend(const AttendArgs& a, hipStream_t st) {
    const Kinds kinds = kinds_of(a);
    AttendArgs m = a;
    hipError_t e = hipSuccess;
    if (kinds.few) {
        const Plan p = plan_attend(a, true);
        m = with_scratch(a, p);
        e = launch_plan(m, p, st);
        if (e == hipSuccess) e = launch_attend_few(m, p.cut, p.items, st);
        if (e == hipSuccess) e = launch_attend_join(m, p.cut, p.tiles, st);
        if (e != hipSuccess || !kinds.many) return e;
        m.parts = (float*)((char*)a.parts + part_bytes(a, p) + plan_bytes(a, p));
    }
    const Plan p = plan_attend(a, false);
    m = with_scratch(m, p);
    if ((e = launch_plan(m, p, st)) != hipSuccess) return e;
    const unsigned grid = p.items * (unsigned)a.pool.kv_heads;
    auto go = [&](auto type, auto dp) {
        constexpr int kType = decltype(type)::value, kDp = decltype(dp)::value;
        if constexpr (kType != kKvI8 || kDp != 96) attend_many_kernel<kType, kDp, kDp <= 128 ? 2 : 1><<<grid, 256, 0, st>>>(m, p.cut);
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
    e = hipGetLastError();
    return e == hipSuccess ? launch_attend_join(m, p.cut, p.tiles, st) : e;
}

// ------------------------------------------------------------------------------------------------- selected pages

namespace {

// A row's pages in pieces of so many blocks that all rows and key heads give about kItems workgroups (at least kLeastBlocks each).
Plan plan_selected(const AttendArgs& a) {
    const int group = a.heads / a.pool.kv_heads, tiles = (group + 15) / 16;
    const int64_t blocks = (int64_t)a.top * (a.pool.page / kKvBlock), all = (int64_t)a.batch.rows * a.pool.kv_heads * tiles;
    int64_t pieces = kItems / all;
    if (pieces > blocks / kLeastBlocks) pieces = blocks / kLeastBlocks;
    if (pieces < 1) pieces = 1;
    const int each = ceil_div(blocks, pieces);
    Plan p{};
    p.cut = Cut{4, 1, 16, ceil_div(blocks, each), each, 1.0f, 0, group, 0, 0, 0};
    p.split = p.cut.target > 1;
    p.tiles = (unsigned)(a.batch.rows * tiles);
    p.items = p.tiles * (unsigned)p.cut.target;
    p.cut.slots = (int)p.items;
    p.cut.tiles = (int)p.tiles;
    return p;
}

}  // namespace

hipError_t launch_select_pages(const AttendArgs& a, hipStream_t st);

size_t attend_selected_scratch(const AttendArgs& a) {
    const Plan p = plan_selected(a);
    return p.split ? part_bytes(a, p) + plan_bytes(a, p) : 0;
}

hipError_t launch_attend_selected(const AttendArgs& a, hipStream_t st) {
    const Plan p = plan_selected(a);
    const AttendArgs m = with_scratch(a, p);
    hipError_t e = launch_select_pages(m, st);
    if (e == hipSuccess) e = launch_attend_few(m, p.cut, p.items, st);
    if (e == hipSuccess && p.split) e = launch_attend_join(m, p.cut, p.tiles, st);
    return e;
}

}  // namespace ovfq
