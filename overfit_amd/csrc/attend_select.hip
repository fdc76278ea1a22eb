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

// A workgroup has `each` pages (a multiple of 64) of a row, from first_row on, and key head. kWhole: heads of 128 or 256 channels.
template <bool kWhole>
__global__ __launch_bounds__(256) void fit_kernel(AttendArgs a, int first_row, int each) {
    extern __shared__ float queries[];  // [group][dim]
    const int kv_heads = a.pool.kv_heads, dim = a.pool.dim, group = a.heads / kv_heads;
    const int row = first_row + (int)(blockIdx.x / (unsigned)kv_heads), head = (int)(blockIdx.x % (unsigned)kv_heads), tid = threadIdx.x;
    const float* q = a.q + ((size_t)row * a.heads + (size_t)head * group) * dim;
    for (int i = tid; i < group * dim; i += 256) queries[i] = q[i];
    __syncthreads();
    const KvRowPlace at = kv_row_place(a.batch, row, a.batch.most);
    if (at.r < 0 || at.place < 0) return;
    const int pages = min(at.place / a.pool.page, a.batch.width), from = (int)blockIdx.y * each;
    if (pages < a.top || from >= pages) return;  // all of them are taken
    uint64_t* out = (uint64_t*)a.fits + (size_t)blockIdx.x * a.batch.width;
    const int part = tid & 3;
    for (int p = from + (tid >> 2); p < min(pages, from + each); p += 64) {
        const int page = page_at(a, at.r, p);
        double best = __builtin_nan("");
        if (page >= 0) {
            const float* s = a.pool.sums + ((size_t)page * kv_heads + head) * dim;
            for (int g0 = 0; g0 < group; g0 += 4) {
                double fit[4] = {0, 0, 0, 0};
                constexpr int kN = kWhole ? 8 : 4;  // loads under way together
                for (int d0 = 4 * part; d0 < dim; d0 += 16 * kN) {
                    f32x4 v[kN];
#pragma unroll
                    for (int k = 0; k < kN; k++) v[k] = kWhole || d0 + 16 * k < dim ? *(const f32x4*)(s + d0 + 16 * k) : f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < kN; k++) {
                        const bool in = kWhole || d0 + 16 * k < dim;
#pragma unroll
                        for (int g = 0; g < 4; g++) {
                            const f32x4 x = in ? *(const f32x4*)(queries + min(g0 + g, group - 1) * dim + d0 + 16 * k) : f32x4{0, 0, 0, 0};
#pragma unroll
                            for (int i = 0; i < 4; i++) fit[g] = fma((double)x[i], (double)v[k][i], fit[g]);
                        }
                    }
                }
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    fit[g] += __shfl_xor(fit[g], 1, 64);
                    fit[g] += __shfl_xor(fit[g], 2, 64);
                    best = fit[g] > best || best != best ? fit[g] : best;
                }
            }
        }
        // (one that is no number fits least: minus infinity is ordered far above 1)
        if (part == 0) out[p] = page < 0 ? 0 : best != best ? 1 : ordered(best + 0.0);
    }
}

constexpr int kBins = 2048, kHeld = 8;  // kHeld: fits a thread keeps in registers

__global__ __launch_bounds__(256) void choose_kernel(AttendArgs a, int first_row) {
    __shared__ int bins[kBins];
    __shared__ int waves[8];
    __shared__ uint32_t differ[8];
    __shared__ int bin_s, left_s;
    const int kv_heads = a.pool.kv_heads, tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int row = first_row + (int)(blockIdx.x / (unsigned)kv_heads), head = (int)(blockIdx.x % (unsigned)kv_heads);
    const KvRowPlace at = kv_row_place(a.batch, row, a.batch.most);
    if (head == 0 && tid == 0) a.where[row] = at.r;
    if (at.r < 0) return;
    const int own = at.place < 0 ? -1 : at.place / a.pool.page;
    const int pages = own < 0 ? 0 : min(own, a.batch.width), need = a.top - 1;
    const uint64_t* fits = (const uint64_t*)a.fits + (size_t)blockIdx.x * a.batch.width;
    const bool all = pages <= need;
    // the last fit taken: those above `bound` in the bits from `shift` on, and of those equal to it there the first `left`
    uint64_t bound = 0;
    int shift = 64, left = need;
    uint64_t held[kHeld];
    // a thread has kHeld neighbouring pages of each 256 * kHeld, the first ones' fits in registers
    auto each_fit = [&](auto f) {
#pragma unroll
        for (int j = 0; j < kHeld; j++) f(held[j]);
        for (int base = 256 * kHeld; base < pages; base += 256 * kHeld)
            for (int p = base + tid * kHeld; p < min(pages, base + (tid + 1) * kHeld); p++) f(fits[p]);
    };
    if (!all && need > 0) {
#pragma unroll
        for (int j = 0; j < kHeld; j++) held[j] = tid * kHeld + j < pages ? fits[tid * kHeld + j] : 0;
        // the bits in which candidates differ: those above are theirs in common
        const uint64_t any = fits[0];  // (0 where page 0 is no candidate: then all bits may differ)
        uint64_t x = 0;
        each_fit([&](uint64_t k) { x |= k ? k ^ any : 0; });
        auto either = [](int p, int q) { return p | q; };
        const uint32_t lo = (uint32_t)wave_join((int)(uint32_t)x, either), hi = (uint32_t)wave_join((int)(uint32_t)(x >> 32), either);
        if (lane == 0) {
            differ[2 * wave] = lo;
            differ[2 * wave + 1] = hi;
        }
        __syncthreads();
        x = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) x |= (uint64_t)differ[2 * i + 1] << 32 | differ[2 * i];
        shift = x ? 64 - __builtin_clzll(x) : 0;
        bound = shift < 64 ? any >> shift << shift : 0;
        while (shift) {
            const int next = shift > 11 ? shift - 11 : 0, width = shift - next;
            for (int i = tid; i < kBins; i += 256) bins[i] = 0;
            __syncthreads();
            each_fit([&](uint64_t k) {
                if (k && (shift == 64 || (k >> shift) == (bound >> shift))) atomicAdd(&bins[(int)(k >> next) & ((1 << width) - 1)], 1);
            });
            __syncthreads();
            // from the top bin down: the bin in which the count reaches `left`
            int mine = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) mine += bins[kBins - 1 - (8 * tid + i)];
            int upto = wave_upto(mine);
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
            const int bin = bin_s, rest = left_s;
            if (bin < 0) {  // fewer candidates than are wanted: all of them
                shift = 0;
                bound = 0;
                left = 0x7fffffff;
                break;
            }
            const bool whole = bins[bin] == rest;
            __syncthreads();
            bound = (shift == 64 ? 0 : bound >> shift << shift) | (uint64_t)bin << next;
            shift = next;
            left = rest;
            if (whole) break;
        }
    }
    int* list = a.chosen + ((size_t)row * kv_heads + head) * a.top;
    int taken = 0, equal = 0;  // so far: listed, and equal to the bound
    if (need > 0) {
        for (int base = 0; base < pages; base += 256 * kHeld) {
            const int first = base + tid * kHeld;
            uint32_t above = 0, same = 0;  // a bit a page
#pragma unroll
            for (int j = 0; j < kHeld; j++) {
                const int p = first + j;
                if (p >= pages) continue;
                if (all) {
                    above |= (uint32_t)(page_at(a, at.r, p) >= 0) << j;
                } else {
                    const uint64_t k = base ? fits[p] : held[j];
                    if (k) {
                        above |= (uint32_t)((k >> shift) > (bound >> shift)) << j;
                        same |= (uint32_t)((k >> shift) == (bound >> shift)) << j;
                    }
                }
            }
            // pages above and equal before this thread's, in one number each of 16 bits
            const int counts = __popc(above) | __popc(same) << 16;
            int upto = wave_upto(counts);
            __syncthreads();
            if (lane == 63) waves[wave] = upto;
            __syncthreads();
            int whole = 0;
            for (int i = 0; i < 4; i++) {
                upto += i < wave ? waves[i] : 0;
                whole += waves[i];
            }
            int rank = equal + ((upto - counts) >> 16);  // of this thread's first equal page
            // of the equal ones the first `left` are taken: so many come before this thread's pages
            int slot = taken + ((upto - counts) & 0xffff) + min(rank, left) - min(equal, left);
#pragma unroll
            for (int j = 0; j < kHeld; j++) {
                const bool equals = same >> j & 1, take = (above >> j & 1) || (equals && rank < left);
                if (take && slot < need) list[slot] = first + j;
                slot += take;
                rank += equals;
            }
            const int equal_now = equal + (whole >> 16);
            taken += (whole & 0xffff) + min(equal_now, left) - min(equal, left);
            equal = equal_now;
        }
    }
    const bool mine = own >= 0 && page_at(a, at.r, own) >= 0;
    for (int i = taken + tid; i < a.top; i += 256) list[i] = mine && i == taken ? own : -1;
}

}  // namespace

// Rows whose fits are kept at a time: all, but no more than kFitBytes of them where that is more than one row (4096 rows of eight key heads
// over tables of 2048 pages would be 537 MB; in four turns of 134 MB they take as long, 5.3 ms with the attention over 16 pages each).
int attend_fit_rows(const AttendArgs& a) {
    constexpr size_t kFitBytes = 128u << 20;
    if (a.top == 1 || a.batch.width < a.top) return 0;  // a row's own page alone, or all of them
    const size_t row = (size_t)a.pool.kv_heads * a.batch.width * sizeof(double), rows = kFitBytes / row;
    return rows >= (size_t)a.batch.rows ? a.batch.rows : rows ? (int)rows : 1;
}

hipError_t launch_select_pages(const AttendArgs& a, hipStream_t st) {
    const int group = a.heads / a.pool.kv_heads, step = a.fit_rows ? a.fit_rows : a.batch.rows;
    for (int first = 0; first < a.batch.rows; first += step) {
        const int count = a.batch.rows - first < step ? a.batch.rows - first : step;
        const unsigned rows = (unsigned)count * (unsigned)a.pool.kv_heads;
        if (a.fit_rows) {
            // 64 pages a workgroup, more where that gives more workgroups than the chip holds at a time
            int each = 64;
            while (each < 512 && (int64_t)rows * a.batch.width / each > 8192) each *= 2;
            const dim3 grid(rows, (unsigned)((a.batch.width + each - 1) / each));
            if (a.pool.dim % 128 == 0)
                fit_kernel<true><<<grid, 256, (size_t)group * a.pool.dim * 4, st>>>(a, first, each);
            else
                fit_kernel<false><<<grid, 256, (size_t)group * a.pool.dim * 4, st>>>(a, first, each);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        choose_kernel<<<rows, 256, 0, st>>>(a, first);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ovfq
