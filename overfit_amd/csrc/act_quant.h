// act_quant.h — the activation quantisers as device functions, for their own launches (quant.hip, q8_mid.hip) and for the launch
// that computes the adapters' low-rank products beside them (adapters.hip). A part is a workgroup of 256 threads.
#pragma once

#include "ovfq_device.h"
#include "ovfq_launch.h"

namespace ovfq {

// Q4KDotKernel.QuantizeActivationQ8K (RT/Q4KDotKernel.cs:71-136): absMax is a max (exact in any order); scale =
// absMax / 127f; inverse = scale > 0 ? 1f / scale : 0f; q = clamp(rint(x * inverse), -127, 127); bsums[g] = sum
// of the 16 quants of group g. Four super-blocks per wave, one per 16-lane DPP row, sixteen consecutive elements (one
// bsum group) per lane: four 16-byte loads and one 16-byte store of quants per lane, the block's absMax by a 4-step
// DPP row max (a wave per block spent most of its time in the 6 cross-lane exchanges of its max).
__device__ __forceinline__ void quantize_q8k_part(int64_t part, const float* __restrict__ x, int64_t n_blocks,
                                                  int8_t* __restrict__ q, float* __restrict__ s, int16_t* __restrict__ bs,
                                                  uint16_t* __restrict__ bh) {
    // wave_id() is a readfirstlane value, so the buffer resource below is provably wave-uniform (SGPRs).
    const int64_t blk0 = (part * 4 + wave_id()) * 4;
    if (blk0 >= n_blocks) return;
    const int lane = threadIdx.x & 63, row = lane >> 4, l16 = lane & 15;
    const int64_t blk = blk0 + row;
    // blocks past the end read zeros (the resource ends with the last block) and store nothing
    const __amdgpu_buffer_rsrc_t xr =
        make_rsrc(x + blk0 * kQK, rsrc_bytes((uint64_t)n_blocks * kQK * 4, (uint64_t)blk0 * kQK * 4));
    float v[16];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const u32x4 t = ld4(xr, (uint32_t)row * 1024u + (uint32_t)l16 * 64u + (uint32_t)i * 16u);
        v[4 * i] = as_float(t.x);
        v[4 * i + 1] = as_float(t.y);
        v[4 * i + 2] = as_float(t.z);
        v[4 * i + 3] = as_float(t.w);
    }
    const Q8KRow r = q8k_quantize_row16(v);
    if (blk < n_blocks) {
        *reinterpret_cast<u32x4*>(q + blk * kQK + l16 * 16) = r.packed;
        bs[blk * 16 + l16] = (int16_t)r.group_sum;
        if (bh) bh[blk * 16 + l16] = __builtin_bit_cast(uint16_t, (_Float16)r.group_sum);
        if (l16 == 0) s[blk] = r.scale;
    }
}

// The same quantisation into operand-ordered planes (launch_quantize_q8k_tiled): the 16-byte piece that lane (g, r16) of
// MFMA t reads goes to byte 1024 t + 256 g + 16 r16 of its (16 rows, super-block) record, so that a wave loads an A operand
// as one contiguous KiB. Piece p of a super-block (elements 16 p ..) belongs to the (t, g) with src_piece(4 t + g) == p of
// the weight format's operand order (Q4KMfma / Q6KMfma). Lane (g, r16) of the min MFMA reads bsums 4 g .. 4 g + 3.
__device__ __forceinline__ void quantize_q8k_tiled_part(int64_t part, const float* __restrict__ x, int64_t n_blocks, int spr,
                                                        int q6, uint8_t* __restrict__ q, uint8_t* __restrict__ s,
                                                        uint8_t* __restrict__ bh) {
    const int64_t blk0 = (part * 4 + wave_id()) * 4;
    if (blk0 >= n_blocks) return;
    const int lane = threadIdx.x & 63, p = lane & 15;
    const int64_t blk = blk0 + (lane >> 4);
    const __amdgpu_buffer_rsrc_t xr =
        make_rsrc(x + blk0 * kQK, rsrc_bytes((uint64_t)n_blocks * kQK * 4, (uint64_t)blk0 * kQK * 4));
    float v[16];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const u32x4 t = ld4(xr, (uint32_t)lane * 64u + (uint32_t)i * 16u);
        v[4 * i] = as_float(t.x);
        v[4 * i + 1] = as_float(t.y);
        v[4 * i + 2] = as_float(t.z);
        v[4 * i + 3] = as_float(t.w);
    }
    const Q8KRow r = q8k_quantize_row16(v);
    if (blk < n_blocks) {
        const int64_t row = blk / spr;
        const size_t rec = (size_t)(row >> 4) * spr + (size_t)(blk - row * spr);
        const int r16 = (int)(row & 15);
        const int slot = tiled_slot(p, q6 != 0);  // 4 t + g
        *reinterpret_cast<u32x4*>(q + rec * kTiledQ + slot * 256 + r16 * 16) = r.packed;
        if (bh)
            *reinterpret_cast<_Float16*>(bh + rec * kTiledB + (p >> 2) * 128 + r16 * 8 + (p & 3) * 2) =
                (_Float16)r.group_sum;
        if (p == 0) *reinterpret_cast<float*>(s + rec * kTiledS + r16 * 4) = r.scale;
    }
}

// Q8DotKernel.Quantize (RT/Q8DotKernel.cs:42-91): 32-element blocks, eight lanes per block.
__device__ __forceinline__ void quantize_q8_0_part(int64_t part, const float* __restrict__ x, int64_t n_blocks,
                                                   int8_t* __restrict__ q, float* __restrict__ s) {
    // One wave covers 8 consecutive blocks; the resource starts at the wave's first block (wave-uniform).
    const int64_t wblk = (part * 4 + wave_id()) * 8;
    const int lane = threadIdx.x & 63;
    const int64_t blk = wblk + (lane >> 3);
    if (wblk >= n_blocks) return;
    const int sub = lane & 7;
    const __amdgpu_buffer_rsrc_t xr = make_rsrc(x + wblk * 32, rsrc_bytes((uint64_t)n_blocks * 128, (uint64_t)wblk * 128));
    const Q80Lane r = q8_0_quantize_lane(ld4(xr, lane * 16));
    if (blk < n_blocks) {
        reinterpret_cast<uint32_t*>(q + blk * 32)[sub] = r.packed;
        if (sub == 0) s[blk] = r.scale;
    }
}

// The same of rows x (planes * plane_in) into the records of q8_mid.hip: eight lanes a block. nb: blocks of a row, wnb: of a
// plane, gph: groups of four of a plane.
__device__ __forceinline__ void quantize_q8_0_tiled_part(int64_t part, const float* __restrict__ x, int64_t n_blocks, int nb,
                                                         int wnb, int gph, uint8_t* __restrict__ q, float* __restrict__ s) {
    const int64_t wblk = (part * 4 + wave_id()) * 8;
    const int lane = threadIdx.x & 63;
    const int64_t blk = wblk + (lane >> 3);
    if (wblk >= n_blocks) return;
    const int sub = lane & 7;  // elements 4 sub .. 4 sub + 3
    const __amdgpu_buffer_rsrc_t xr = make_rsrc(x + wblk * 32, rsrc_bytes((uint64_t)n_blocks * 128, (uint64_t)wblk * 128));
    const Q80Lane r = q8_0_quantize_lane(ld4(xr, lane * 16));
    if (blk >= n_blocks) return;
    const int64_t row = blk / nb;
    const int b = (int)(blk - row * nb), plane = b / wnb, bp = b - plane * wnb;
    const int64_t rec = (row >> 4) * ((int64_t)(nb / wnb) * gph) + plane * gph + bp / 4;
    const int j = bp & 3, r16 = (int)(row & 15), g = sub >> 1;
    uint8_t* dst = q + rec * 2048 + (j >> 1) * 1024 + (g * 16 + r16) * 16 + (j & 1) * 8 + (sub & 1) * 4;
    *reinterpret_cast<uint32_t*>(dst) = r.packed;
    if (sub == 0) s[rec * 64 + j * 16 + r16] = r.scale;
}

// One of the four, by the job's kind (wave-uniform).
__device__ __forceinline__ void quantize_part(const ActQuantJob& j, int64_t part) {
    if (j.kind == ActQuantJob::kQ8K)
        quantize_q8k_part(part, j.x, j.n_blocks, j.q, j.s, j.b, j.bh);
    else if (j.kind == ActQuantJob::kQ8KTiled)
        quantize_q8k_tiled_part(part, j.x, j.n_blocks, j.per_row, j.q6, reinterpret_cast<uint8_t*>(j.q),
                                reinterpret_cast<uint8_t*>(j.s), j.q6 ? nullptr : reinterpret_cast<uint8_t*>(j.bh));
    else if (j.kind == ActQuantJob::kQ80)
        quantize_q8_0_part(part, j.x, j.n_blocks, j.q, j.s);
    else if (j.kind == ActQuantJob::kQ80Tiled)
        quantize_q8_0_tiled_part(part, j.x, j.n_blocks, j.per_row, j.per_row, (j.per_row + 3) / 4,
                                 reinterpret_cast<uint8_t*>(j.q), j.s);
}

}  // namespace ovfq
