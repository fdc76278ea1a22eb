// adapters.hip — low-rank adapters of many requests beside a shared projection: for every activation row m with an adapter
// slot s, y[m] += scale_s * B_s (A_s x[m]), A_s [rank][in], B_s [out][rank].
//
// Two launches behind the projection's: the rows' low-rank products A_s x[m] into a scratch plane, then B_s times them into the
// outputs. Products and sums are fp32 whatever the adapters are kept in.
#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

namespace {

template <int kType>
__device__ __forceinline__ float value_at(const void* p, int64_t i) {
    if constexpr (kType == kAdapterF32) return static_cast<const float*>(p)[i];
    const uint16_t u = static_cast<const uint16_t*>(p)[i];
    if constexpr (kType == kAdapterF16) return half_bits_to_float(u);
    return as_float((uint32_t)u << 16);
}

// The slot of row m, or -1 for a row without an adapter (no such slot, or none loaded there).
__device__ __forceinline__ int slot_of(const AdapterJob& j, const int* row_slots, int m) {
    const int s = row_slots[m];
    return s >= 0 && s < j.slots && j.info[s].rank > 0 ? s : -1;
}

// grid (rows, jobs): a wave per rank index in turn, its lanes along the inputs.
template <int kType>
__global__ __launch_bounds__(256) void adapter_shrink_kernel(const AdapterArgs a) {
    const AdapterJob j = a.job[blockIdx.y];
    const int m = blockIdx.x;
    const int s = slot_of(j, a.row_slots, m);
    if (s < 0) return;
    const int rank = j.info[s].rank, lane = threadIdx.x & 63;
    const float* x = a.x + (int64_t)m * a.in;
    for (int r = threadIdx.x >> 6; r < rank; r += 4) {
        const int64_t base = ((int64_t)s * j.max_rank + r) * a.in;
        float sum = 0.0f;
        for (int k = lane; k < a.in; k += 64) sum = fmaf(x[k], value_at<kType>(j.a, base + k), sum);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if (lane == 0) j.low[(int64_t)m * j.max_rank + r] = sum;
    }
}

// grid (rows, output tiles of 256, jobs): a thread per output.
template <int kType>
__global__ __launch_bounds__(256) void adapter_expand_kernel(const AdapterArgs a) {
    const AdapterJob j = a.job[blockIdx.z];
    const int n = blockIdx.y * 256 + threadIdx.x, m = blockIdx.x;
    const int s = slot_of(j, a.row_slots, m);
    if (s < 0 || n >= j.out) return;
    const int rank = j.info[s].rank;
    const float* low = j.low + (int64_t)m * j.max_rank;
    const int64_t base = (int64_t)s * j.out * j.b_stride + (int64_t)n * rank_pad(rank);
    float sum = 0.0f;
    for (int r = 0; r < rank; r++) sum = fmaf(low[r], value_at<kType>(j.b, base + r), sum);
    float* y = j.y + (int64_t)m * j.out + n;
    *y = fmaf(sum, j.info[s].scale, *y);
}

__global__ void adapter_slot_kernel(AdapterSlot* info, int slot, int rank, float scale) {
    info[slot] = AdapterSlot{rank, scale};
}

// B [out][rank] -> rows of rank_pad(rank) values, zeros past the rank. T: the values' storage width.
template <class T>
__global__ __launch_bounds__(256) void adapter_pad_kernel(const T* __restrict__ src, T* __restrict__ dst, int64_t n, int rank,
                                                          int pad) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t row = i / pad;
    const int r = (int)(i - row * pad);
    dst[i] = r < rank ? src[row * rank + r] : T(0);
}

template <int kType>
hipError_t launch_apply(const AdapterArgs& a, int jobs, hipStream_t st) {
    int out = 0;
    for (int i = 0; i < jobs; i++) out = a.job[i].out > out ? a.job[i].out : out;
    hipLaunchKernelGGL(adapter_shrink_kernel<kType>, dim3((unsigned)a.rows, (unsigned)jobs), dim3(256), 0, st, a);
    hipLaunchKernelGGL(adapter_expand_kernel<kType>, dim3((unsigned)a.rows, (unsigned)((out + 255) / 256), (unsigned)jobs),
                       dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_adapters(const AdapterArgs& a, int type, int jobs, hipStream_t st) {
    if (type == kAdapterF32) return launch_apply<kAdapterF32>(a, jobs, st);
    if (type == kAdapterF16) return launch_apply<kAdapterF16>(a, jobs, st);
    return launch_apply<kAdapterBF16>(a, jobs, st);
}

hipError_t launch_adapter_slot(AdapterSlot* info, int slot, int rank, float scale, hipStream_t st) {
    hipLaunchKernelGGL(adapter_slot_kernel, dim3(1), dim3(1), 0, st, info, slot, rank, scale);
    return hipGetLastError();
}

hipError_t launch_adapter_pad(const void* src, void* dst, int out, int rank, int elem, hipStream_t st) {
    const int pad = rank_pad(rank);
    const int64_t n = (int64_t)out * pad;
    const dim3 grid((unsigned)((n + 255) / 256));
    if (elem == 4)
        hipLaunchKernelGGL(adapter_pad_kernel<uint32_t>, grid, dim3(256), 0, st, (const uint32_t*)src, (uint32_t*)dst, n, rank,
                           pad);
    else
        hipLaunchKernelGGL(adapter_pad_kernel<uint16_t>, grid, dim3(256), 0, st, (const uint16_t*)src, (uint16_t*)dst, n, rank,
                           pad);
    return hipGetLastError();
}

}  // namespace ovfq
