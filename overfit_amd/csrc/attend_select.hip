// attend_select.hip — the pages that a row's queries fit best, before attention over them alone.
//
//   fit(page) = max over the key head's query heads of q . (sum of the page's keys)
//
// over the full pages before the row's own; of these the best `top` - 1 (of equal fits the lower page), and the row's own page. Fits
// are fp64 products and sums of fp32 operands: which side of the border a page falls on does not depend on an order of additions.
//
// Bound: HBM, each full page's sum (4 dim bytes) once for its request's rows and key head. Four lanes a page, 64 pages a workgroup at a
// time, queries in LDS. The choice is a radix search for the last fit taken, eleven bits a step over the ordered bits of the fits,
// which ends when a step's bin is taken whole (two or three steps), then a pass that lists the pages in rising order.
#include "attend.h"

namespace ovfq {

namespace {

constexpr int kFitPages = 256;  // pages a workgroup

struct RowPlace {
    int r, place;
};
// The row's request (the first that has it), or -1, and its token's place.
__device__ __forceinline__ RowPlace row_place(const KvBatch& b, int row, int* found) {
    if (threadIdx.x == 0) *found = b.requests;
    __syncthreads();
    for (int r = threadIdx.x; r < b.requests; r += 256) {
        const KvRows m = kv_rows(b, r);
        if (m.n && m.n <= b.most && row >= m.first && row < m.first + m.n) atomicMin(found, r);
    }
    __syncthreads();
    const int r = __builtin_amdgcn_readfirstlane(*found);
    if (r >= b.requests) return RowPlace{-1, -1};
    const KvRows m = kv_rows(b, r);
    return RowPlace{r, kv_length(b, r) - m.n + (row - m.first)};
}

__device__ __forceinline__ int page_at(const AttendArgs& a, int r, int entry) {
    if (entry < 0 || entry >= a.batch.width) return -1;
    const int p = a.batch.tables[(size_t)r * a.batch.width + entry];
    return p >= 0 && p < a.pool.pages ? p : -1;
}

// Doubles as unsigned integers of the same order; 0 is none of them.
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return u >> 63 ? ~u : u | 1ull << 63;
}

__global__ __launch_bounds__(256) void fit_kernel(AttendArgs a) {
    extern __shared__ float queries[];  // [group][dim]
    __shared__ int found;
    const int kv_heads = a.pool.kv_heads, dim = a.pool.dim, group = a.heads / kv_heads;
    const int row = (int)(blockIdx.x / (unsigned)kv_heads), head = (int)(blockIdx.x % (unsigned)kv_heads), tid = threadIdx.x;
    const RowPlace at = row_place(a.batch, row, &found);
    if (at.r < 0 || at.place < 0) return;
    const int pages = min(at.place / a.pool.page, a.batch.width), from = (int)blockIdx.y * kFitPages;
    if (pages < a.top || from >= pages) return;  // all of them are taken
    const float* q = a.q + ((size_t)row * a.heads + (size_t)head * group) * dim;
    for (int i = tid; i < group * dim; i += 256) queries[i] = q[i];
    __syncthreads();
    uint64_t* out = (uint64_t*)a.fits + ((size_t)row * kv_heads + head) * a.batch.width;
    const int part = tid & 3;
    for (int p = from + (tid >> 2); p < min(pages, from + kFitPages); p += 64) {
        const int page = page_at(a, at.r, p);
        double best = -__builtin_inf();
        if (page >= 0) {
            const float* s = a.pool.sums + ((size_t)page * kv_heads + head) * dim;
            for (int g0 = 0; g0 < group; g0 += 4) {
                double fit[4] = {0, 0, 0, 0};
                for (int d = 4 * part; d < dim; d += 16) {
                    const f32x4 v = *(const f32x4*)(s + d);
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const f32x4 x = *(const f32x4*)(queries + min(g0 + g, group - 1) * dim + d);
#pragma unroll
                        for (int i = 0; i < 4; i++) fit[g] = fma((double)x[i], (double)v[i], fit[g]);
                    }
                }
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    fit[g] += __shfl_xor(fit[g], 1, 64);
                    fit[g] += __shfl_xor(fit[g], 2, 64);
                    best = fit[g] > best ? fit[g] : best;  // (one that is no number fits least)
                }
            }
        }
        if (part == 0) out[p] = page >= 0 ? ordered(best + 0.0) : 0;
    }
}

constexpr int kBins = 2048;

__global__ __launch_bounds__(256) void choose_kernel(AttendArgs a) {
    __shared__ int bins[kBins];
    __shared__ int waves[8];
    __shared__ int found, bin_s, left_s;
    const int kv_heads = a.pool.kv_heads, tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int row = (int)(blockIdx.x / (unsigned)kv_heads), head = (int)(blockIdx.x % (unsigned)kv_heads);
    const RowPlace at = row_place(a.batch, row, &found);
    if (head == 0 && tid == 0) a.where[row] = at.r;
    if (at.r < 0) return;
    const int own = at.place < 0 ? -1 : at.place / a.pool.page;
    const int pages = own < 0 ? 0 : min(own, a.batch.width), need = a.top - 1;
    const uint64_t* fits = (const uint64_t*)a.fits + ((size_t)row * kv_heads + head) * a.batch.width;
    const bool all = pages <= need;
    // the last fit taken: those above `bound` in the bits from `shift` on, and of those equal to it there the first `left`
    uint64_t bound = 0;
    int shift = 64, left = need;
    if (!all && need > 0) {
        for (;;) {
            const int next = shift >= 20 ? shift - 11 : 0, width = shift - next;
            for (int i = tid; i < kBins; i += 256) bins[i] = 0;
            __syncthreads();
            for (int p = tid; p < pages; p += 256) {
                const uint64_t k = fits[p];
                if (k && (shift == 64 || (k >> shift) == (bound >> shift))) atomicAdd(&bins[(int)(k >> next) & ((1 << width) - 1)], 1);
            }
            __syncthreads();
            // from the top bin down: the bin in which the count reaches `left`
            int mine = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) mine += bins[kBins - 1 - (8 * tid + i)];
            int upto = mine;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int v = __shfl_up(upto, off, 64);
                if (lane >= off) upto += v;
            }
            if (lane == 63) waves[wave] = upto;
            if (tid == 0) bin_s = -1;
            __syncthreads();
            for (int i = 0; i < wave; i++) upto += waves[i];
            if (upto >= left && upto - mine < left) {
                int rest = left - (upto - mine), i = 0;
                for (;; i++) {
                    const int n = bins[kBins - 1 - (8 * tid + i)];
                    if (rest <= n) break;
                    rest -= n;
                }
                bin_s = kBins - 1 - (8 * tid + i);
                left_s = rest;
            }
            __syncthreads();
            const int bin = bin_s;
            const int rest = left_s;
            if (bin < 0) {  // fewer candidates than are wanted: all of them
                shift = 64;
                left = 0x7fffffff;
                break;
            }
            const bool whole = bins[bin] == rest;
            __syncthreads();
            bound = (shift == 64 ? 0 : bound >> shift << shift) | (uint64_t)bin << next;
            shift = next;
            left = rest;
            if (whole || shift == 0) break;
        }
    }
    int* list = a.chosen + ((size_t)row * kv_heads + head) * a.top;
    int taken = 0, equal = 0;  // so far: listed, and equal to the bound
    if (need > 0) {
        for (int base = 0; base < pages; base += 256) {
            const int p = base + tid;
            bool above = false, same = false;
            if (p < pages) {
                if (all) {
                    above = page_at(a, at.r, p) >= 0;
                } else {
                    const uint64_t k = fits[p];
                    if (k && shift == 64) above = true;
                    else if (k) {
                        above = (k >> shift) > (bound >> shift);
                        same = (k >> shift) == (bound >> shift);
                    }
                }
            }
            const uint64_t before = (1ull << lane) - 1;
            uint64_t votes = __ballot(same);
            if (lane == 0) waves[wave] = __popcll(votes);
            __syncthreads();
            int rank = equal + __popcll(votes & before);
            for (int i = 0; i < 4; i++) {
                rank += i < wave ? waves[i] : 0;
                equal += waves[i];
            }
            const bool take = above || (same && rank < left);
            votes = __ballot(take);
            if (lane == 0) waves[4 + wave] = __popcll(votes);
            __syncthreads();
            int slot = taken + __popcll(votes & before);
            for (int i = 0; i < 4; i++) {
                slot += i < wave ? waves[4 + i] : 0;
                taken += waves[4 + i];
            }
            if (take && slot < need) list[slot] = p;
            __syncthreads();
        }
    }
    const bool mine = own >= 0 && page_at(a, at.r, own) >= 0;
    for (int i = taken + tid; i < a.top; i += 256) list[i] = mine && i == taken ? own : -1;
}

}  // namespace

hipError_t launch_select_pages(const AttendArgs& a, hipStream_t st) {
    const int group = a.heads / a.pool.kv_heads;
    const unsigned rows = (unsigned)a.batch.rows * (unsigned)a.pool.kv_heads;
    if (a.batch.width >= a.top && a.top > 1) {
        fit_kernel<<<dim3(rows, (unsigned)((a.batch.width + kFitPages - 1) / kFitPages)), 256, (size_t)group * a.pool.dim * 4, st>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    choose_kernel<<<rows, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace ovfq
