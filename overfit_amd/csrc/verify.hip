// verify.hip — verification of drafted tokens against the target model's logits, with given random numbers.
//
// A request's rows of logits are the target's answers after its last token and after each of its n drafted tokens. With
// p_i = softmax(logits_i / temperature) (temperature not above 0: all of it on the first largest logit) and q_i the
// distribution that draft i was drawn from (none given: all of it on the draft itself), draft i is accepted while
// u_i q_i(x_i) < p_i(x_i). The first draft refused is replaced by a draw from max(p_i - q_i, 0), or, with none refused, a token
// is drawn from p_n: the smallest token whose running sum of the weights passes u times their total. Accepted and drawn
// tokens together are then distributed as the target alone would draw them.
//
// Probabilities, totals and running sums are fp64: among 128256 running sums in fp32 a hundredth of all draws would land in
// the rounding of a neighbour. An exponential is a power of two, a table's 2^(j / 128) and a polynomial of the rest (table-driven
// range reduction as Tang published it in 1989), within 2.5e-12 of its value: 10 fp64 instructions a token, where the library's exp()
// made the first launch take 37.7 us on 240 rows of 128256 instead of 24.7 (5.0 TB/s, a large copy's rate).
//
// Two launches. (1) A wave per row and 2048 tokens: the largest logit and the sum of exponentials relative to it. (2) A
// workgroup per request: a wave a row joins the row's sums and decides the draft, the first refused wins; the sums of the row to
// draw from are its pieces' weights already (a one-hot q takes its token's away), so that only the piece that the draw falls into
// is read again. With the drafts' distributions the weights are max(p - q, 0) of all tokens: then a workgroup per request and
// two pieces, and the last of a request to finish, by a counter, draws.
#include <cmath>

#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

namespace {

constexpr int kPiece = kVerifyPiece;
constexpr int kHalf = kPiece / 2;  // a wave of the first launch
constexpr int kThreads = 256;      // of the first launch
constexpr int kSpan = 2;       // pieces a workgroup of the second sums up
constexpr int kDrawThreads = 512, kDrawWaves = kDrawThreads / 64;

// v of the lane that the DPP control names, `none` where there is no such lane: within 16 lanes (row_shr 1, 2, 4, 8), then the last
// lane of the row before (row_bcast15) and of the 32 before (row_bcast31). Six steps scan a wave, some 10 cycles each, where a
// shuffle goes through LDS.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t from_lane(uint32_t v, uint32_t none) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, kCtrl, kRows, 0xf, false);
}
template <int kCtrl, int kRows>
__device__ __forceinline__ double from_lane(double v) {  // + 0 where there is none
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = from_lane<kCtrl, kRows>((uint32_t)b, 0u), hi = from_lane<kCtrl, kRows>((uint32_t)(b >> 32), 0u);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane),
                   hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// The sum over the lanes up to this one.
__device__ __forceinline__ double wave_scan(double v) {
    v += from_lane<0x111, 0xf>(v);
    v += from_lane<0x112, 0xf>(v);
    v += from_lane<0x114, 0xf>(v);
    v += from_lane<0x118, 0xf>(v);
    v += from_lane<0x142, 0xa>(v);
    v += from_lane<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) { return lane_of(wave_scan(v), 63); }

template <class Op>
__device__ __forceinline__ uint32_t wave_join(uint32_t v, uint32_t none, Op op) {
    v = op(v, from_lane<0x111, 0xf>(v, none));
    v = op(v, from_lane<0x112, 0xf>(v, none));
    v = op(v, from_lane<0x114, 0xf>(v, none));
    v = op(v, from_lane<0x118, 0xf>(v, none));
    v = op(v, from_lane<0x142, 0xa>(v, none));
    v = op(v, from_lane<0x143, 0xc>(v, none));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_max(float v) {
    return as_float(wave_join(__builtin_bit_cast(uint32_t, v), 0xff800000u, [](uint32_t x, uint32_t y) {
        return __builtin_bit_cast(uint32_t, fmaxf(as_float(x), as_float(y)));
    }));
}
__device__ __forceinline__ int wave_min(int v) {
    return (int)wave_join((uint32_t)v, 0x7fffffffu, [](uint32_t x, uint32_t y) { return (uint32_t)min((int)x, (int)y); });
}

// A NaN logit counts as -inf (the token has no probability).
__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : v; }

__device__ __forceinline__ bool is_greedy(float temperature) { return !(temperature > 0.0f && temperature < INFINITY); }

// Exponentials of non-positive numbers. With z = x 128 / ln2 = n + f, n the nearest whole number, exp(x) = 2^(n / 128) 2^(f / 128);
// the second factor is the Taylor polynomial of degree 3 of f ln2 / 128, |.| <= 0.0028, off by its fourth power / 24 < 2.5e-12. n
// comes out of the low bits of a sum with 1.5 * 2^52. The table has 2^(j / 128), j < 128, less j << 13 in the high word, so that
// n << 13 added to it puts the whole 2^(n / 128) together. (Running sums of 128256 probabilities that are off by 2.5e-12 each, now
// up, now down, move a draw to a neighbour once in 10^8.)
constexpr int kPowers = 128;
constexpr double kMagic = 6755399441055744.0, kPer = 128 / 0.69314718055994530942;  // 1.5 * 2^52, 128 / ln2
__device__ __forceinline__ void fill_powers(u32x2* powers) {  // a barrier comes before their use
    const uint32_t j = threadIdx.x;
    if (j >= (uint32_t)kPowers) return;
    const u32x2 v = __builtin_bit_cast(u32x2, exp2((double)j * (1.0 / kPowers)));
    powers[j] = u32x2{v.x, v.y - (j << 13)};
}
__device__ __forceinline__ double small_power(double f) {  // 2^(f / 128)
    constexpr double c = 0.69314718055994530942 / 128;
    return fma(f, fma(f, fma(f, c * c * c / 6, c * c / 2), c), 1.0);
}
__device__ __forceinline__ double whole_power(uint32_t n, const u32x2* powers) {  // 2^(n / 128) in the normal range
    const u32x2 v = powers[n & (kPowers - 1)];
    return __builtin_bit_cast(double, u32x2{v.x, v.y + (n << 13)});
}
__device__ __forceinline__ uint32_t low_word(double t) { return __builtin_bit_cast(u32x2, t).x; }
// sum + exp(d per ln2 / 128), d <= 0; floor: the d of exp(-700), below which it is 1e-304, which no sum with a 1 in it sees.
__device__ __forceinline__ double add_exp(double sum, double d, double per, double floor, const u32x2* powers) {
    d = fmax(d, floor);
    const double t = fma(d, per, kMagic);
    const double f = fma(d, per, kMagic - t);
    return fma(whole_power(low_word(t), powers), small_power(f), sum);
}
// exp(x), x <= 0, right below the normal range too: 0 in the end.
__device__ __forceinline__ double negative_exp(double x, const u32x2* powers) {
    x = fmax(x, -800.0);
    const double t = fma(x, kPer, kMagic);
    const uint32_t n = low_word(t);
    return ldexp(whole_power(n & (kPowers - 1), powers) * small_power(fma(x, kPer, kMagic - t)), (int)n >> 7);
}

// Tokens lo + 4 (i * kT + t) .. + 3, i < kN / 4, of a row of `vocab`; past the row `fill`.
template <int kT, int kN>
__device__ __forceinline__ void load_tokens(const float* row, int vocab, int lo, int t, float fill, float (&v)[kN]) {
    const int n = min(kT * kN, vocab - lo);
    const __amdgpu_buffer_rsrc_t r = make_rsrc(row + lo, (uint32_t)n * 4);
    u32x4 raw[kN / 4];
#pragma unroll
    for (int i = 0; i < kN / 4; i++) raw[i] = ld4(r, 16u * (uint32_t)(i * kT + t));
#pragma unroll
    for (int i = 0; i < kN / 4; i++) {
        const uint32_t a[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int c = 0; c < 4; c++) v[4 * i + c] = as_float(a[c]);
    }
    if (n == kT * kN) return;
#pragma unroll
    for (int i = 0; i < kN; i++)
        if (4 * ((i >> 2) * kT + t) + (i & 3) >= n) v[i] = fill;
}

// The request that owns `row` (its offsets in order and within the rows), or -1; the same for every lane of the wave.
__device__ __forceinline__ int owner_of(const VerifyArgs& a, int row) {
    int owner = -1;
    for (int r0 = 0; r0 < a.requests; r0 += 64) {
        const int r = r0 + (int)(threadIdx.x & 63);
        bool mine = false;
        if (r < a.requests) {
            const int lo = a.row_offsets[r], hi = a.row_offsets[r + 1];
            mine = lo >= 0 && lo <= row && row < hi && hi <= a.rows;
        }
        const uint64_t at = __ballot(mine);
        if (at) owner = r0 + 63 - __builtin_clzll(at);
    }
    return owner;
}

__global__ __launch_bounds__(kThreads, 8) void verify_stats_kernel(const VerifyArgs a) {
    constexpr int kEach = kHalf / 64;
    __shared__ u32x2 powers[kPowers];
    const int row = (int)(blockIdx.z * gridDim.y + blockIdx.y), half = (int)blockIdx.x * (kThreads / 64) + wave_id();
    const int lane = threadIdx.x & 63, lo = half * kHalf;
    if (row >= a.rows) return;
    fill_powers(powers);
    __syncthreads();
    if (a.done && !row && !blockIdx.x)
        for (int r = threadIdx.x; r < a.requests; r += kThreads) a.done[r] = 0;
    if (half >= 2 * a.pieces) return;
    VerifyStat out{-INFINITY, 0x7fffffff, 0.0};
    if (lo < a.vocab) {
        float v[kEach];
        load_tokens<64>(a.logits + (int64_t)row * a.vocab, a.vocab, lo, lane, -INFINITY, v);
        const int request = owner_of(a, row);
        if (request < 0) return;
        const float temperature = a.temperature ? a.temperature[request] : 1.0f;
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kEach; i++) m = fmaxf(m, v[i]);  // (passes over NaN, as add_exp's maximum does)
        out.max = m = wave_max(m);
        if (is_greedy(temperature)) {
            int at = 0x7fffffff;
#pragma unroll
            for (int i = kEach - 1; i >= 0; i--)
                if (v[i] == m) at = lo + 4 * ((i >> 2) * 64 + lane) + (i & 3);
            out.at = wave_min(at);
        } else if (m > -INFINITY && m < INFINITY) {
            const double per = kPer / (double)temperature, floor = -700.0 * (double)temperature;
            double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
            for (int i = 0; i < kEach; i++) s[i & 3] = add_exp(s[i & 3], (double)v[i] - (double)m, per, floor, powers);
            out.sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
        }
    }
    if (lane == 0) a.stats[(int64_t)row * 2 * a.pieces + half] = out;
}

struct Pair {
    VerifyStat half[2];
};
__device__ __forceinline__ Pair load_pair(const VerifyArgs& a, int row, int piece) {
    return *reinterpret_cast<const Pair*>(a.stats + ((int64_t)row * a.pieces + piece) * 2);
}
// A piece's sum relative to `most`.
__device__ __forceinline__ double sum_of(const Pair& p, float most, double inv, const u32x2* powers) {
    double sum = 0.0;
#pragma unroll
    for (int h = 0; h < 2; h++)
        if (p.half[h].sum > 0.0) sum += p.half[h].sum * negative_exp(((double)p.half[h].max - (double)most) * inv, powers);
    return sum;
}

// A row's pieces joined by one wave: the largest logit, its first token, and the sum of exponentials relative to it. first: the
// lane's piece; mine: its sum relative to the row's largest.
__device__ __forceinline__ VerifyStat join_row(const VerifyArgs& a, int row, double inv, const u32x2* powers, const Pair& first,
                                               double& mine) {
    const int lane = threadIdx.x & 63;
    float m = fmaxf(first.half[0].max, first.half[1].max);
    for (int c = 64 + lane; c < a.pieces; c += 64) {
        const Pair v = load_pair(a, row, c);
        m = fmaxf(m, fmaxf(v.half[0].max, v.half[1].max));
    }
    m = wave_max(m);
    auto first_of = [&](const Pair& p) { return p.half[0].max == m ? p.half[0].at : p.half[1].max == m ? p.half[1].at : 0x7fffffff; };
    int at = first_of(first);
    double sum = mine = sum_of(first, m, inv, powers);
    for (int c = 64 + lane; c < a.pieces; c += 64) {
        const Pair v = load_pair(a, row, c);
        at = min(at, first_of(v));
        sum += sum_of(v, m, inv, powers);
    }
    return VerifyStat{m, wave_min(at), wave_sum(sum)};
}

__device__ __forceinline__ bool has_distribution(const VerifyStat& s) { return s.max > -INFINITY && s.max < INFINITY; }

// A piece's sum as the weight to draw it by. Below the normal range a token's weight may round to zero where its piece's does not: a
// piece whose largest logit, `most`, weighs nothing has no token to draw.
constexpr double kNormal = 1e-290;  // a 4096th of it, divided by a row's sum of up to 2^31, is in the normal range still
__device__ __forceinline__ double drawable(double sum, float most, const VerifyStat& s, double inv, const u32x2* powers) {
    if (sum >= kNormal || sum == 0.0) return sum;
    return negative_exp(((double)most - (double)s.max) * inv, powers) * (1.0 / s.sum) > 0.0 ? sum : 0.0;
}

// The sum over the workgroup, to every thread.
__device__ __forceinline__ double block_sum(double v, double* shared) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kDrawWaves; w++) s += shared[w];
    return s;
}

// Bound by the chain of dependent reads: the offsets, the rows' sums and the drafts' values, the piece to draw from.
template <bool kProbs>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(const VerifyArgs a) {
    constexpr int kEach = kPiece / kDrawThreads;
    __shared__ u32x2 powers[kPowers];
    __shared__ double shared[kDrawWaves], totals[kSpan > kEach / 4 ? kSpan : kEach / 4][kDrawWaves];
    __shared__ int first, found, last;
    __shared__ VerifyStat drawn;
    __shared__ double pieces[64], chance;  // of the row to draw from: the first pieces' sums, and p of its draft
    __shared__ float tops[kProbs ? 64 : 1];  // and their largest logits
    const int r = (int)(blockIdx.z * gridDim.y + blockIdx.y), piece = (int)blockIdx.x * kSpan;
    if (r >= a.requests) return;
    const int t = threadIdx.x, wave = wave_id(), lane = t & 63;
    const int row0 = a.row_offsets[r], end = a.row_offsets[r + 1];
    const float temperature = a.temperature ? a.temperature[r] : 1.0f, final_u = a.final_uniforms[r];
    fill_powers(powers);
    if (row0 < 0 || end <= row0 || end > a.rows) {  // no such request
        if (piece == 0 && t == 0) a.accepted[r] = -1;
        return;
    }
    const int n = end - row0 - 1;
    const bool greedy = is_greedy(temperature);
    const double inv = greedy ? 0.0 : 1.0 / (double)temperature;
    if (t == 0) {
        first = n;
        found = 0x7fffffff;
        last = -1;
    }
    __syncthreads();
    // the first row that a wave does not keep; row n, behind the last draft, is none's to keep
    int kept = 0x7fffffff;
    VerifyStat s{};
    double mine = 0.0, p = 0.0;  // the lane's piece, and the draft's chance
    float most = -INFINITY;      // the piece's largest logit
    for (int i = wave; i <= n; i += kDrawWaves) {
        const int d = row0 - r + i;  // draft i of the request among all drafts
        const bool draft = i < n && d >= 0 && d < a.drafts;
        const VerifyStat none{-INFINITY, 0x7fffffff, 0.0};
        Pair own{{none, none}};
        if (lane < a.pieces) own = load_pair(a, row0 + i, lane);
        int x = -1;
        float logit = 0.0f, q = 1.0f, u = 0.0f;
        if (draft) {
            x = a.draft_tokens[d];
            u = a.accept_uniforms[d];
            if (x >= 0 && x < a.vocab) {
                logit = clean(a.logits[(int64_t)(row0 + i) * a.vocab + x]);
                if (kProbs) q = fmaxf(a.draft_probs[(int64_t)d * a.vocab + x], 0.0f);
            }
        }
        s = join_row(a, row0 + i, inv, powers, own, mine);
        most = fmaxf(own.half[0].max, own.half[1].max);
        bool ok = false;
        p = 0.0;
        if (x >= 0 && x < a.vocab && has_distribution(s)) {
            p = greedy ? (x == s.at ? 1.0 : 0.0) : negative_exp(((double)logit - (double)s.max) * inv, powers) / s.sum;
            ok = (double)u * (double)q < p;
        }
        if (!ok) {
            kept = i;
            break;
        }
    }
    if (kept < n && lane == 0) atomicMin(&first, kept);
    __syncthreads();
    if (kept == first) {
        // (with probabilities later, where a piece is asked for: 16 requests 28.1 us so, 27.2; without, one request 15.3 later, 14.4)
        pieces[lane] = kProbs ? mine : drawable(mine, most, s, inv, powers);
        if (kProbs) tops[lane] = most;
        if (lane == 0) {
            drawn = s;
            chance = p;
        }
    }
    kept = first;
    __syncthreads();
    s = drawn;
    const int row = row0 + kept, d = row0 - r + kept;
    if (piece == 0) {
        if (t == 0) a.accepted[r] = kept;
        for (int i = t; i <= n; i += kDrawThreads)
            if (i != kept) a.tokens[row0 + i] = i < kept ? a.draft_tokens[row0 - r + i] : -1;
    }
    if (greedy || !has_distribution(s)) {  // without q's part of it the weight is on one token still
        if (piece == 0 && t == 0) a.tokens[row] = has_distribution(s) ? s.at : -1;
        return;
    }
    bool rest = kept < n && d >= 0 && d < a.drafts;  // draw from max(p - q, 0)
    const double scale = 1.0 / s.sum;
    const float* logits = a.logits + (int64_t)row * a.vocab;
    const float* probs = kProbs && rest ? a.draft_probs + (int64_t)d * a.vocab : nullptr;
    const int x = !kProbs && rest ? a.draft_tokens[d] : -1;
    auto weight = [&](float logit, float q) {
        const double p = negative_exp(((double)clean(logit) - (double)s.max) * inv, powers) * scale;
        return kProbs && rest ? fmax(p - (double)fmaxf(q, 0.0f), 0.0) : p;
    };
    double* parts = a.parts + (int64_t)r * a.pieces;
    if (kProbs && rest) {
        float v[kSpan][kEach], q[kSpan][kEach];
#pragma unroll
        for (int h = 0; h < kSpan; h++) {  // (past the last piece: that one again, unused)
            const int lo = min(piece + h, a.pieces - 1) * kPiece;
            load_tokens<kDrawThreads>(logits, a.vocab, lo, t, -INFINITY, v[h]);
            load_tokens<kDrawThreads>(probs, a.vocab, lo, t, 0.0f, q[h]);
        }
        double sum[kSpan];
#pragma unroll
        for (int h = 0; h < kSpan; h++) {
            sum[h] = 0.0;
#pragma unroll
            for (int i = 0; i < kEach; i++) sum[h] += weight(v[h][i], q[h][i]);
            sum[h] = wave_sum(sum[h]);
            if (lane == 0) totals[h][wave] = sum[h];
        }
        __syncthreads();
        // the last of the request's workgroups sees all parts: each is stored before its workgroup counts itself
        if (t == 0) {
#pragma unroll
            for (int h = 0; h < kSpan; h++) {
                double all = 0.0;
#pragma unroll
                for (int o = 0; o < kDrawWaves; o++) all += totals[h][o];
                if (piece + h < a.pieces) __hip_atomic_store(parts + piece + h, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            first = __hip_atomic_fetch_add(a.done + r, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (first != (int)gridDim.x - 1) return;
    } else if (piece) {
        return;
    }
    // The pieces' weights: the parts, or from the rows' sums, without the draft's own.
    double alone = -1.0;  // the weight of the draft's piece
    auto of_piece = [&](int c) {
        if (c >= a.pieces) return 0.0;
        if (kProbs && rest) return __hip_atomic_load(parts + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (c == x / kPiece && alone >= 0.0) return alone;
        if (c < 64) return (kProbs ? drawable(pieces[c], tops[c], s, inv, powers) : pieces[c]) * scale;
        const Pair v = load_pair(a, row, c);
        return drawable(sum_of(v, s.max, inv, powers), fmaxf(v.half[0].max, v.half[1].max), s, inv, powers) * scale;
    };
    if (!kProbs && x >= 0 && x < a.vocab) {
        const double all = of_piece(x / kPiece), left = all - chance;
        if (all > kNormal && left > 1e-3 * all) {
            alone = left;
        } else {  // too little is left for a difference, or for the others to have a weight each: the sum of the others
            float v[kEach];
            load_tokens<kDrawThreads>(logits, a.vocab, x / kPiece * kPiece, t, -INFINITY, v);
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < kEach; i++)
                sum += x / kPiece * kPiece + 4 * ((i >> 2) * kDrawThreads + t) + (i & 3) == x ? 0.0 : weight(v[i], 0.0f);
            alone = block_sum(sum, shared);
        }
    }
    auto add_up = [&] {
        double sum = of_piece(lane);
        for (int c = 64 + lane; c < a.pieces; c += 64) sum += of_piece(c);
        return wave_sum(sum);
    };
    double total = add_up();
    bool whole = false;
    if (rest && !(total > 0.0)) {  // nothing left of p beside q: draw from p
        rest = false;
        whole = true;
        alone = -1.0;
        total = add_up();
    }
    // (a number of 1 or more: no running sum passes the total, also not one that rounding puts above it)
    const double target = final_u < 1.0f ? (double)final_u * total : INFINITY;
    // the piece in which the running sum passes (every wave the same)
    double before = 0.0, some_before = 0.0;
    int hit = -1, some = 0;
    for (int c0 = 0; c0 < a.pieces && hit < 0; c0 += 64) {
        const double w = of_piece(c0 + lane), upto = before + wave_scan(w);
        const uint64_t any = __ballot(w > 0.0), over = __ballot(w > 0.0 && upto > target);
        if (any) {
            const int l = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
            some = c0 + l;
            some_before = l ? lane_of(upto, l - 1) : before;
            if (over) hit = some;
        }
        before = lane_of(upto, 63);
    }
    // rounding at the very end: the last token with a weight
    const int lo = some * kPiece;
    float v[kEach], q[kEach];
    load_tokens<kDrawThreads>(logits, a.vocab, lo, t, -INFINITY, v);
    if (kProbs && rest) load_tokens<kDrawThreads>(probs, a.vocab, lo, t, 0.0f, q);
    // four tokens a thread and stretch of 4 kDrawThreads
    constexpr int kStretches = kEach / 4;
    double w[kEach], fours[kStretches], upto[kStretches];
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const int token = lo + 4 * ((i >> 2) * kDrawThreads + t) + (i & 3);
        w[i] = token < a.vocab && (whole || token != x) ? weight(v[i], kProbs && rest ? q[i] : 0.0f) : 0.0;
        fours[i >> 2] = i & 3 ? fours[i >> 2] + w[i] : w[i];
    }
#pragma unroll
    for (int i = 0; i < kStretches; i++) {
        upto[i] = wave_scan(fours[i]);
        if (lane == 63) totals[i][wave] = upto[i];
    }
    __syncthreads();
    int at = 0x7fffffff, behind = -1;
    double prior = some_before;
#pragma unroll
    for (int i = 0; i < kStretches; i++) {
        double sum = prior + (upto[i] - fours[i]);
#pragma unroll
        for (int o = 0; o < kDrawWaves; o++) {
            const double other = totals[i][o];
            if (o < wave) sum += other;
            prior += other;
        }
#pragma unroll
        for (int c = 0; c < 4; c++) {
            sum += w[4 * i + c];
            if (w[4 * i + c] > 0.0) {
                behind = lo + 4 * (i * kDrawThreads + t) + c;
                if (sum > target && at == 0x7fffffff) at = behind;
            }
        }
    }
    if (at != 0x7fffffff) atomicMin(&found, at);
    if (behind >= 0) atomicMax(&last, behind);
    __syncthreads();
    if (t == 0) a.tokens[row] = found != 0x7fffffff ? found : last;
}

}  // namespace

hipError_t launch_verify_drafts(const VerifyArgs& a, hipStream_t st) {
    auto grid = [](int x, int n) {  // n in two dimensions
        const unsigned y = (unsigned)(n < 65535 ? n : 65535);
        return dim3((unsigned)x, y, ((unsigned)n + y - 1) / y);
    };
    hipLaunchKernelGGL(verify_stats_kernel, grid((2 * a.pieces + kThreads / 64 - 1) / (kThreads / 64), a.rows), dim3(kThreads), 0, st, a);
    if (a.draft_probs)
        hipLaunchKernelGGL(verify_draw_kernel<true>, grid((a.pieces + kSpan - 1) / kSpan, a.requests), dim3(kDrawThreads), 0, st, a);
    else
        hipLaunchKernelGGL(verify_draw_kernel<false>, grid(1, a.requests), dim3(kDrawThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace ovfq
