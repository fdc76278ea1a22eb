// norm.hip — the step between two blocks of a transformer in one pass over the rows:
//   t = post(y);  h' = h + scale * gate * t;  x = pre(h')
// with RMS or layer norms: n(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps) * weight + bias, the means over the row, no mean
// subtracted and no bias in the RMS form. Sums, variances and the two planes are fp32. Layer norms sum up the differences from the
// fp32 mean and their squares together, and take the mean that is left out of both: a mean of 10^4 standard deviations would be up to
// 2 * 10^-3 of them off by itself, which all elements of the row would have in common. (us, two layer norms, without that / with:
// 1 row of 4096 4.5 / 4.8, 512 rows 9.3 / 9.6, 2048 rows 30.3 / 30.3, 1024 rows of 8192 30.5 / 31.9, 400 of 20480 92.6 / 94.7.)
//
// Bound: HBM for many rows (each input element is read once and each output written once; a row stays in registers between its
// two norms), launch and two dependent reductions for one. A group of kT threads owns a row: 16 to 64 lanes for rows of up to
// 512 elements (several rows a workgroup, sums by lane exchanges alone), two to sixteen waves for rows of up to 16384, and past
// that a workgroup that reads the row once per step.
#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

__device__ __forceinline__ f32x4 ldf4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(f32x4, ld4(r, off));
}

// Sum over the kT threads that own a row; every one of them receives it. kT > 64: `red` holds a float per wave, in two halves
// that successive sums of a row alternate between (one barrier a sum).
template <int kT>
__device__ __forceinline__ float group_sum(float v, float* red, int& turn) {
#pragma unroll
    for (int off = (kT < 64 ? kT : 64) / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    if constexpr (kT > 64) {
        constexpr int kW = kT / 64;
        float* half = red + 2 * kW * (turn & 1);
        turn++;
        if ((threadIdx.x & 63) == 0) half[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < kW; i++) v += half[i];
    }
    return v;
}

// Two sums in the exchange of one; `red` holds two floats per wave and half.
template <int kT>
__device__ __forceinline__ void group_sums(float& v, float& w, float* red, int& turn) {
#pragma unroll
    for (int off = (kT < 64 ? kT : 64) / 2; off >= 1; off >>= 1) {
        v += __shfl_xor(v, off, 64);
        w += __shfl_xor(w, off, 64);
    }
    if constexpr (kT > 64) {
        constexpr int kW = kT / 64;
        float* half = red + 2 * kW * (turn & 1);
        turn++;
        if ((threadIdx.x & 63) == 0) {
            half[threadIdx.x >> 6] = v;
            half[kW + (threadIdx.x >> 6)] = w;
        }
        __syncthreads();
        v = w = 0.0f;
#pragma unroll
        for (int i = 0; i < kW; i++) {
            v += half[i];
            w += half[kW + i];
        }
    }
}

// (a maximum would turn NaN, which stays in all of its row, into 0)
__device__ __forceinline__ float not_below_0(float v) { return v < 0.0f ? 0.0f : v; }

// A side's weights and biases for the thread's pieces.
template <int kT, int kNV>
struct Side {
    f32x4 w[kNV], b[kNV];
    __device__ __forceinline__ void load(const NormSide& n, int k, int t) {
        const __amdgpu_buffer_rsrc_t wr = make_rsrc(n.weight, n.weight ? (uint32_t)k * 4 : 0u);
        const __amdgpu_buffer_rsrc_t br = make_rsrc(n.bias, n.bias ? (uint32_t)k * 4 : 0u);
#pragma unroll
        for (int i = 0; i < kNV; i++) w[i] = ldf4(wr, 16u * (uint32_t)(t + i * kT));
        if (n.bias) {
#pragma unroll
            for (int i = 0; i < kNV; i++) b[i] = ldf4(br, 16u * (uint32_t)(t + i * kT));
        }
    }
};

// The norm of one row of k elements held as kNV four-element pieces a thread; elements past the row are zero and stay out of
// the sums. kLate: the side is loaded here, not before.
template <int kT, int kNV, bool kLate>
__device__ __forceinline__ void norm_row(f32x4 (&v)[kNV], Side<kT, kNV>& side, const NormSide& n, int k, int t, float* red,
                                         int& turn) {
    const float inv_k = 1.0f / (float)k;
    float s = 0.0f, rest = 0.0f, var = 0.0f;
    auto centre = [&] {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kNV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) sum += v[i][c];
        const float mean = group_sum<kT>(sum, red, turn) * inv_k;
#pragma unroll
        for (int i = 0; i < kNV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                v[i][c] = 4 * (t + i * kT) + c < k ? v[i][c] - mean : 0.0f;
                rest += v[i][c];
            }
    };
    auto squares = [&] {
#pragma unroll
        for (int i = 0; i < kNV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) s = fmaf(v[i][c], v[i][c], s);
    };
    auto centred = [&] {
        group_sums<kT>(s, rest, red, turn);
        rest *= inv_k;
        var = not_below_0(fmaf(-rest, rest, s * inv_k));
#pragma unroll
        for (int i = 0; i < kNV; i++) v[i] -= rest;  // (what is past the row is not used)
    };
    if constexpr (kT == 1024 && kNV == 4) {
        // One code for both norms' squares where the registers are short (us, RMS, one / two: 16384 wide, 512 rows 30.4 / 34.3; 4096
        // wide, 2048 rows 28.4 / 27.6)
        if (n.layer) centre();
        squares();
        if (n.layer)
            centred();
        else
            var = group_sum<kT>(s, red, turn) * inv_k;
    } else if (n.layer) {
        centre();
        squares();
        centred();
    } else {
        squares();
        var = group_sum<kT>(s, red, turn) * inv_k;
    }
    const float r = 1.0f / sqrtf(var + n.eps);
    if (!kLate) {
#pragma unroll
        for (int i = 0; i < kNV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                v[i][c] *= r;
                if (n.weight) v[i][c] *= side.w[i][c];
                if (n.bias) v[i][c] += side.b[i][c];
            }
        return;
    }
    // piece by piece
    const __amdgpu_buffer_rsrc_t wr = make_rsrc(n.weight, n.weight ? (uint32_t)k * 4 : 0u);
    const __amdgpu_buffer_rsrc_t br = make_rsrc(n.bias, n.bias ? (uint32_t)k * 4 : 0u);
#pragma unroll
    for (int i = 0; i < kNV; i++) v[i] *= r;
    if (n.weight) {
#pragma unroll
        for (int i = 0; i < kNV; i++) v[i] *= ldf4(wr, 16u * (uint32_t)(t + i * kT));
    }
    if (n.bias) {
#pragma unroll
        for (int i = 0; i < kNV; i++) v[i] += ldf4(br, 16u * (uint32_t)(t + i * kT));
    }
}

template <int kT, int kNV>
__device__ __forceinline__ void store_row(float* p, const f32x4 (&v)[kNV], int k, int t) {
#pragma unroll
    for (int i = 0; i < kNV; i++) {
        const int e = 4 * (t + i * kT);
        if (e + 4 <= k) {
            __builtin_memcpy(p + e, &v[i], 16);  // a row starts on any 4-byte boundary
        } else {
#pragma unroll
            for (int c = 0; c < 3; c++)
                if (e + c < k) p[e + c] = v[i][c];
        }
    }
}

// Rows of up to 4 * kT * kNV elements. Everything that the row needs is loaded before its first sum; kLate: the weights and the
// gate only where they are used, so that twice the waves fit the registers.
template <int kT, int kNV, bool kLate>
__global__ __launch_bounds__(kT <= 64 ? 256 : kT, !kLate ? 1 : kNV == 4 && kT < 1024 ? 6 : 8) void residual_norm_kernel(const NormArgs a) {
    constexpr int kRows = kT <= 64 ? 256 / kT : 1;  // rows a workgroup
    __shared__ float red[kT > 64 ? 4 * (kT / 64) : 1];
    const int t = kRows > 1 ? (int)threadIdx.x % kT : (int)threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * kRows;
    const int sub = kRows > 1 ? (int)threadIdx.x / kT : 0;
    const int64_t row = row0 + sub;
    const int k = a.k;
    int turn = 0;
    // one resource over the workgroup's rows: what is past a row's end is masked below, what is past the last row reads zeros
    const int64_t left = a.rows - row0 < kRows ? a.rows - row0 : kRows;
    const uint32_t bytes = (uint32_t)left * (uint32_t)k * 4;
    const uint32_t base = (uint32_t)sub * (uint32_t)k * 4;
    f32x4 v[kNV], h[kNV], g[kNV];
    Side<kT, kNV> post, pre;
    auto load_plane = [&](const float* p, f32x4(&d)[kNV]) {
        const __amdgpu_buffer_rsrc_t r = make_rsrc(p + row0 * k, bytes);
#pragma unroll
        for (int i = 0; i < kNV; i++) d[i] = ldf4(r, base + 16u * (uint32_t)(t + i * kT));
    };
    auto load_gate = [&] {
        if (a.gate_mode == kGateFull) {
            load_plane(a.gate, g);
        } else if (a.gate_mode == kGateChannel) {
            const __amdgpu_buffer_rsrc_t r = make_rsrc(a.gate, (uint32_t)k * 4);
#pragma unroll
            for (int i = 0; i < kNV; i++) g[i] = ldf4(r, 16u * (uint32_t)(t + i * kT));
        }
    };
    load_plane(a.y, v);
    constexpr bool kLateH = kLate && kT == 1024 && kNV == 4;  // (does not fit the registers of two workgroups a CU)
    if (a.h && !kLateH) load_plane(a.h, h);
    float g_row = a.scale;
    if (a.gate_mode == kGateRow) {
        const __amdgpu_buffer_rsrc_t r = make_rsrc(a.gate + row0, (uint32_t)left * 4);
        g_row *= as_float(ld1(r, (uint32_t)sub * 4));
    }
    if (!kLate) {
        if (a.has_post) post.load(a.post, k, t);
        load_gate();
        if (a.has_pre) pre.load(a.pre, k, t);
    }
#pragma unroll
    for (int i = 0; i < kNV; i++)
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (4 * (t + i * kT) + c >= k) v[i][c] = 0.0f;
    if (a.has_post) norm_row<kT, kNV, kLate>(v, post, a.post, k, t, red, turn);
    if (kLate) load_gate();
    if (a.gate_mode == kGateFull || a.gate_mode == kGateChannel) {
#pragma unroll
        for (int i = 0; i < kNV; i++) v[i] *= g[i];
    }
    if (a.h && kLateH) load_plane(a.h, h);
#pragma unroll
    for (int i = 0; i < kNV; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float s = v[i][c] * g_row;
            v[i][c] = 4 * (t + i * kT) + c < k ? (a.h ? h[i][c] + s : s) : 0.0f;
        }
    const bool live = row < a.rows;
    if (a.h_out && live) store_row<kT, kNV>(a.h_out + row * k, v, k, t);
    if (!a.has_pre) return;
    norm_row<kT, kNV, kLate>(v, pre, a.pre, k, t, red, turn);
    if (live) store_row<kT, kNV>(a.x_out + row * k, v, k, t);
}

// Rows past 16384 elements: a workgroup of 1024 reads its row once per sum and once more for x (from the caches, where a row of
// that length still lies). h_out may be the h plane and x_out the y plane: each element is read by the thread that writes it,
// and the last step reads h' back from h_out where there is one.
__global__ __launch_bounds__(1024) void residual_norm_long_kernel(const NormArgs a) {
    __shared__ float red[64];
    const int64_t row = blockIdx.x;
    const int k = a.k, t = threadIdx.x;
    const float* y = a.y + row * k;
    const float* h = a.h ? a.h + row * k : nullptr;
    float* ho = a.h_out ? a.h_out + row * k : nullptr;
    const float inv_k = 1.0f / (float)k;
    int turn = 0;
    struct Stats {
        float mean, rest, r;  // (two means to take out: together they have more digits than one has)
    };
    auto stats = [&](const NormSide& n, auto&& at) {
        float s = 0.0f;
        if (!n.layer) {
            for (int e = t; e < k; e += 1024) {
                const float d = at(e);
                s = fmaf(d, d, s);
            }
            return Stats{0.0f, 0.0f, 1.0f / sqrtf(group_sum<1024>(s, red, turn) * inv_k + n.eps)};
        }
        for (int e = t; e < k; e += 1024) s += at(e);
        const float mean = group_sum<1024>(s, red, turn) * inv_k;
        float rest = s = 0.0f;
        for (int e = t; e < k; e += 1024) {
            const float d = at(e) - mean;
            s = fmaf(d, d, s);
            rest += d;
        }
        group_sums<1024>(s, rest, red, turn);
        rest *= inv_k;
        return Stats{mean, rest, 1.0f / sqrtf(not_below_0(fmaf(-rest, rest, s * inv_k)) + n.eps)};
    };
    auto apply = [](const NormSide& n, float v, int e, const Stats& s) {
        v = ((v - s.mean) - s.rest) * s.r;
        if (n.weight) v *= n.weight[e];
        return n.bias ? v + n.bias[e] : v;
    };
    Stats post{0.0f, 0.0f, 1.0f};
    if (a.has_post) post = stats(a.post, [&](int e) { return y[e]; });
    const float g_row = a.gate_mode == kGateRow ? a.scale * a.gate[row] : a.scale;
    auto sum_at = [&](int e) {
        float v = a.has_post ? apply(a.post, y[e], e, post) : y[e];
        if (a.gate_mode == kGateFull) v *= a.gate[row * k + e];
        if (a.gate_mode == kGateChannel) v *= a.gate[e];
        v *= g_row;
        return h ? h[e] + v : v;
    };
    if (ho)
        for (int e = t; e < k; e += 1024) ho[e] = sum_at(e);
    if (!a.has_pre) return;
    float* x = a.x_out + row * k;
    if (ho) {  // an element is read back by the thread that wrote it
        const Stats pre = stats(a.pre, [&](int e) { return ho[e]; });
        for (int e = t; e < k; e += 1024) x[e] = apply(a.pre, ho[e], e, pre);
    } else {
        const Stats pre = stats(a.pre, sum_at);
        for (int e = t; e < k; e += 1024) x[e] = apply(a.pre, sum_at(e), e, pre);
    }
}

template <int kT, int kNV, bool kLate>
hipError_t launch(const NormArgs& a, hipStream_t st) {
    constexpr int kRows = kT <= 64 ? 256 / kT : 1;
    hipLaunchKernelGGL((residual_norm_kernel<kT, kNV, kLate>), dim3((unsigned)((a.rows + kRows - 1) / kRows)),
                       dim3(kT <= 64 ? 256 : kT), 0, st, a);
    return hipGetLastError();
}

}  // namespace

// Two pieces a thread and all loads first up to 2048 elements (the 161 registers of four pieces so leave three waves a SIMD); past
// that the weights late (us, two norms, residual, channel gate, all first with four pieces / late with four / late with two:
// 4096 wide 1 row 3.9 / 3.8 / 3.4, 512 rows 7.5 / 6.9 / 6.8, 1024 rows 14.7 / 12.7 / 12.9, 2048 rows 29.0 / 28.6 / 29.5; 2049 wide
// 3000 rows 25.0 / 21.9 / 23.3; 8192 wide 1 row 4.5 / 4.3 / 4.2, 1024 rows 34.6 / 30.8 / 29.0; 1024 wide 64 rows 3.8 / 3.7 / 3.2, 8192
// rows 27.9 / 28.2 / 27.3; 16384 wide 1 row 13.8 / 6.6, 512 rows 53.5 / 30.4; two pieces, first / late: 2048 wide 1 row 3.1 / 3.2, 4096 rows
// 27.4 / 28.1; 512 wide 16384 rows 26.4 / 27.0). At 26 to 29 us these planes of 134 MB move at 4.6 to 5.1 TB/s, a large copy's rate.
hipError_t launch_residual_norm(const NormArgs& a, hipStream_t st) {
    const int k = a.k;
    if (k <= 64) return launch<16, 1, false>(a, st);
    if (k <= 128) return launch<32, 1, false>(a, st);
    if (k <= 256) return launch<64, 1, false>(a, st);
    if (k <= 512) return launch<64, 2, false>(a, st);
    if (k <= 1024) return launch<128, 2, true>(a, st);
    if (k <= 2048) return launch<256, 2, false>(a, st);
    if (k <= 4096) return a.rows > 1024 ? launch<256, 4, true>(a, st) : launch<512, 2, true>(a, st);
    if (k <= 8192) return launch<1024, 2, true>(a, st);
    if (k <= 16384) return launch<1024, 4, true>(a, st);
    hipLaunchKernelGGL(residual_norm_long_kernel, dim3((unsigned)a.rows), dim3(1024), 0, st, a);
    return hipGetLastError();
}

}  // namespace ovfq
