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
// the rounding of a neighbour. Bound: reading the logits once (HBM), and the fp64 exponentials behind it.
//
// Three launches. (1) A workgroup per row and 8192 tokens: the largest logit and the sum of exponentials relative to it.
// (2) A workgroup per request and 8192 tokens: the rows' sums joined, the drafts decided (every workgroup of a request repeats
// this, it takes less than a launch), and the weights of its tokens in the row to draw from summed. (3) A workgroup per
// request: the piece, then the token in it, where the running sum passes.
#include <cmath>

#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int kPiece = kVerifyPiece;  // tokens a workgroup: 256 threads x 8 four-token loads
constexpr int kThreads = 256;
constexpr int kVecs = kPiece / (4 * kThreads);

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
    return v;
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = min(v, __shfl_xor(v, off, 64));
    return v;
}

// A NaN logit counts as -inf (the token has no probability).
__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : v; }

__device__ __forceinline__ bool is_greedy(float temperature) { return !(temperature > 0.0f && temperature < INFINITY); }

// Tokens [lo, lo + kPiece) of a row of `vocab`: piece i of a thread is tokens lo + 4 (i * kThreads + t) on; past the row
// `fill`.
__device__ __forceinline__ void load_piece(const float* row, int vocab, int lo, int t, float fill, float (&v)[4 * kVecs]) {
    const int n = min(kPiece, vocab - lo);
    const __amdgpu_buffer_rsrc_t r = make_rsrc(row + lo, (uint32_t)n * 4);
    u32x4 raw[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; i++) raw[i] = ld4(r, 16u * (uint32_t)(i * kThreads + t));
#pragma unroll
    for (int i = 0; i < kVecs; i++) {
        const uint32_t a[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int c = 0; c < 4; c++) v[4 * i + c] = 4 * (i * kThreads + t) + c < n ? as_float(a[c]) : fill;
    }
}

// The request that owns `row` (its offsets in order and within the rows), or -1; every thread of the workgroup calls it.
__device__ __forceinline__ int owner_of(const VerifyArgs& a, int row, int* shared) {
    if (threadIdx.x == 0) *shared = -1;
    __syncthreads();
    for (int r = threadIdx.x; r < a.requests; r += kThreads) {
        const int lo = a.row_offsets[r], hi = a.row_offsets[r + 1];
        if (lo >= 0 && lo <= row && row < hi && hi <= a.rows) atomicMax(shared, r);
    }
    __syncthreads();
    return *shared;
}

__global__ __launch_bounds__(kThreads) void verify_stats_kernel(const VerifyArgs a) {
    __shared__ int owner;
    __shared__ float wmax[4];
    __shared__ double wsum[4];
    __shared__ int wmin[4];
    const int row = (int)blockIdx.x / a.pieces, piece = (int)blockIdx.x % a.pieces;
    const int t = threadIdx.x, wave = t >> 6, lo = piece * kPiece;
    float v[4 * kVecs];
    load_piece(a.logits + (int64_t)row * a.vocab, a.vocab, lo, t, -INFINITY, v);
    const int request = owner_of(a, row, &owner);
    if (request < 0) return;
    const float temperature = a.temperature ? a.temperature[request] : 1.0f;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * kVecs; i++) {
        v[i] = clean(v[i]);
        m = fmaxf(m, v[i]);
    }
    m = wave_max(m);
    if ((t & 63) == 0) wmax[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    VerifyStat out{m, 0x7fffffff, 0.0};
    if (is_greedy(temperature)) {
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 4 * kVecs - 1; i >= 0; i--)
            if (v[i] == m) at = lo + 4 * ((i >> 2) * kThreads + t) + (i & 3);
        at = wave_min(at);
        if ((t & 63) == 0) wmin[wave] = at;
        __syncthreads();
        out.at = min(min(wmin[0], wmin[1]), min(wmin[2], wmin[3]));
    } else if (m > -INFINITY && m < INFINITY) {
        const double inv = 1.0 / (double)temperature;
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 4 * kVecs; i++) s += exp(((double)v[i] - (double)m) * inv);
        s = wave_sum(s);
        if ((t & 63) == 0) wsum[wave] = s;
        __syncthreads();
        out.sum = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
    }
    if (t == 0) a.stats[(int64_t)row * a.pieces + piece] = out;
}

// A row's pieces joined by one wave: the largest logit, its first token, and the sum of exponentials relative to it.
__device__ __forceinline__ VerifyStat join_row(const VerifyArgs& a, int row, double inv) {
    const VerifyStat* s = a.stats + (int64_t)row * a.pieces;
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int c = lane; c < a.pieces; c += 64) m = fmaxf(m, s[c].max);
    m = wave_max(m);
    int at = 0x7fffffff;
    double sum = 0.0;
    for (int c = lane; c < a.pieces; c += 64) {
        if (s[c].max == m) at = min(at, s[c].at);
        if (s[c].sum > 0.0) sum += s[c].sum * exp(((double)s[c].max - (double)m) * inv);
    }
    return VerifyStat{m, wave_min(at), wave_sum(sum)};
}

// p of one token from its row's joined sums.
__device__ __forceinline__ double prob(float logit, int token, const VerifyStat& s, bool greedy, double inv) {
    if (greedy) return token == s.at ? 1.0 : 0.0;
    return exp(((double)clean(logit) - (double)s.max) * inv) / s.sum;
}

__device__ __forceinline__ bool has_distribution(const VerifyStat& s) { return s.max > -INFINITY && s.max < INFINITY; }

__global__ __launch_bounds__(kThreads) void verify_decide_kernel(const VerifyArgs a) {
    __shared__ int refused;
    __shared__ double wsum[4], wrest[4];
    const int r = (int)blockIdx.x / a.pieces, piece = (int)blockIdx.x % a.pieces;
    const int t = threadIdx.x, wave = t >> 6;
    const int row0 = a.row_offsets[r], end = a.row_offsets[r + 1];
    if (row0 < 0 || end <= row0 || end > a.rows) {
        if (piece == 0 && t == 0) {
            a.accepted[r] = -1;
            a.pick[r].row = -1;
        }
        return;
    }
    const int n = end - row0 - 1;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = is_greedy(temperature);
    const double inv = greedy ? 0.0 : 1.0 / (double)temperature;
    if (t == 0) refused = n;
    __syncthreads();
    for (int i = wave; i < n; i += 4) {
        const VerifyStat s = join_row(a, row0 + i, inv);
        const int d = row0 - r + i;  // draft i of the request among all drafts
        bool ok = false;
        if (d >= 0 && d < a.drafts && has_distribution(s)) {
            const int x = a.draft_tokens[d];
            if (x >= 0 && x < a.vocab) {
                const double p = prob(a.logits[(int64_t)(row0 + i) * a.vocab + x], x, s, greedy, inv);
                const float q = a.draft_probs ? fmaxf(a.draft_probs[(int64_t)d * a.vocab + x], 0.0f) : 1.0f;
                ok = (double)a.accept_uniforms[d] * (double)q < p;
            }
        }
        if (!ok && (t & 63) == 0) atomicMin(&refused, i);
    }
    __syncthreads();
    const int kept = refused;
    const int row = row0 + kept;
    const VerifyStat s = join_row(a, row, inv);
    const int d = row0 - r + kept;
    const bool rest = kept < n && d >= 0 && d < a.drafts;  // draw from max(p - q, 0)
    if (piece == 0) {
        if (t == 0) {
            a.accepted[r] = kept;
            a.pick[r] = VerifyPick{row, rest ? d : -1, s};
        }
        for (int i = t; i <= n; i += kThreads)
            if (i != kept) a.tokens[row0 + i] = i < kept ? a.draft_tokens[row0 - r + i] : -1;
    }
    const int lo = piece * kPiece;
    double sum = 0.0, left = 0.0;
    if (has_distribution(s)) {
        float v[4 * kVecs], q[4 * kVecs];
        load_piece(a.logits + (int64_t)row * a.vocab, a.vocab, lo, t, -INFINITY, v);
        const int x = rest && !a.draft_probs ? a.draft_tokens[d] : -1;
        if (rest && a.draft_probs) load_piece(a.draft_probs + (int64_t)d * a.vocab, a.vocab, lo, t, 0.0f, q);
#pragma unroll
        for (int i = 0; i < 4 * kVecs; i++) {
            const int token = lo + 4 * ((i >> 2) * kThreads + t) + (i & 3);
            const double p = token < a.vocab ? prob(v[i], token, s, greedy, inv) : 0.0;
            sum += p;
            if (rest && a.draft_probs)
                left += fmax(p - (double)fmaxf(q[i], 0.0f), 0.0);
            else
                left += token == x ? 0.0 : p;
        }
    }
    sum = wave_sum(sum);
    left = wave_sum(left);
    if ((t & 63) == 0) {
        wsum[wave] = sum;
        wrest[wave] = left;
    }
    __syncthreads();
    if (t == 0) {
        double* part = a.parts + 2 * ((int64_t)r * a.pieces + piece);
        part[0] = (wrest[0] + wrest[1]) + (wrest[2] + wrest[3]);
        part[1] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
    }
}

__global__ __launch_bounds__(kThreads) void verify_pick_kernel(const VerifyArgs a) {
    __shared__ double run[kThreads];
    __shared__ int found, last;
    const int r = blockIdx.x, t = threadIdx.x;
    const VerifyPick pk = a.pick[r];
    if (pk.row < 0) return;
    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = is_greedy(temperature);
    const double inv = greedy ? 0.0 : 1.0 / (double)temperature;
    const double* part = a.parts + 2 * (int64_t)r * a.pieces;
    // the totals of both weights, and the piece that the draw falls into (every thread the same)
    double total = 0.0, total_p = 0.0;
    for (int c = 0; c < a.pieces; c++) {
        total += part[2 * c];
        total_p += part[2 * c + 1];
    }
    const bool rest = pk.draft >= 0 && total > 0.0;  // nothing left of p beside q: draw from p
    if (!rest) total = total_p;
    if (!(total > 0.0)) {  // no finite logit
        if (t == 0) a.tokens[pk.row] = -1;
        return;
    }
    const double target = (double)a.final_uniforms[r] * total;
    double before = 0.0;
    int piece = -1, some = 0;
    double at_some = 0.0;
    for (int c = 0; c < a.pieces && piece < 0; c++) {
        const double w = part[2 * c + (rest ? 0 : 1)];
        if (w > 0.0) {
            some = c;
            at_some = before;
            if (before + w > target) piece = c;
        }
        before += w;
    }
    if (piece < 0) piece = some;  // rounding at the very end: the last token with a weight
    before = at_some;
    // 32 consecutive tokens a thread
    constexpr int kEach = kPiece / kThreads;
    const int lo = piece * kPiece + t * kEach;
    const float* lg = a.logits + (int64_t)pk.row * a.vocab;
    const float* q = rest && a.draft_probs ? a.draft_probs + (int64_t)pk.draft * a.vocab : nullptr;
    const int x = rest && !a.draft_probs ? a.draft_tokens[pk.draft] : -1;
    double w[kEach], mine = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const int token = lo + i;
        double p = 0.0;
        if (token < a.vocab) {
            p = prob(lg[token], token, pk.stat, greedy, inv);
            if (q) p = fmax(p - (double)fmaxf(q[token], 0.0f), 0.0);
            if (token == x) p = 0.0;
        }
        w[i] = p;
        mine += p;
    }
    if (t == 0) {
        found = 0x7fffffff;
        last = -1;
    }
    run[t] = mine;
    __syncthreads();
    double sum = before;
    for (int i = 0; i < t; i++) sum += run[i];
    int hit = 0x7fffffff, mine_last = -1;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        sum += w[i];
        if (w[i] > 0.0) {
            if (sum > target && hit == 0x7fffffff) hit = lo + i;
            mine_last = lo + i;
        }
    }
    if (hit != 0x7fffffff) atomicMin(&found, hit);
    if (mine_last >= 0) atomicMax(&last, mine_last);
    __syncthreads();
    if (t == 0) a.tokens[pk.row] = found != 0x7fffffff ? found : last;
}

}  // namespace

hipError_t launch_verify_drafts(const VerifyArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(verify_stats_kernel, dim3((unsigned)a.rows * (unsigned)a.pieces), dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL(verify_decide_kernel, dim3((unsigned)a.requests * (unsigned)a.pieces), dim3(kThreads), 0, st, a);
    hipLaunchKernelGGL(verify_pick_kernel, dim3((unsigned)a.requests), dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace ovfq
