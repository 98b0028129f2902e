// One thread's share of an attention softmax on tensor memory: scores of 64 columns of its row, masks, weights (the prefill kernels).
#pragma once

#include "prefill_tc_common.cuh"

namespace vq {

using namespace ptx;

constexpr float kT4Lazy = 8.f;    // log2 units: P stays below 2^8

// scores of 64 columns outside [lo, hi) of the step: excluded
__device__ __forceinline__ void t4_mask_range(uint32_t (&r)[64], int lo, int hi)
{
#pragma unroll
    for (int c = 0; c < 64; ++c)
        if (c < lo || c >= hi) r[c] = 0xff800000u;
}

// Far tile with empty codes: a code with cnt == 0 is excluded from the maximum and from P, as the reference does before its
// maximum (ops/triton_fused_vq_attn.py:44-46) - otherwise an unused codeword with a dominating score could push every real
// weight below the exponent range.  cw: the counts of the step's 64 columns.
__device__ __forceinline__ void t4_mask_empty(uint32_t (&r)[64], const float *cw)
{
#pragma unroll
    for (int c = 0; c < 64; c += 4) {
        const float4 w = *reinterpret_cast<const float4 *>(cw + c);
        if (!(w.x > 0.f)) r[c] = 0xff800000u;
        if (!(w.y > 0.f)) r[c + 1] = 0xff800000u;
        if (!(w.z > 0.f)) r[c + 2] = 0xff800000u;
        if (!(w.w > 0.f)) r[c + 3] = 0xff800000u;
    }
}

__device__ __forceinline__ float t4_max(const uint32_t (&r)[64])
{
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 32; ++j) mx[j & 3] = fmax3(mx[j & 3], __uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// P = exp2(S * scale - m) of the 64 scores, packed 16-bit floats (the tensor pipe's operands) written to the 32 columns at p_addr; returns
// sum plus the (FAR: count-weighted) sums of the two halves, one after the other.
template <bool FAR, bool F16>
__device__ __forceinline__ float t4_exp(const uint32_t (&r)[64], uint32_t p_addr, const float *cw, float scale_log2, float neg_m, float sum)
{
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = 32 * half + 4 * j;
            float w[4] = {1.f, 1.f, 1.f, 1.f};
            if (FAR) {
                const float4 w4 = *reinterpret_cast<const float4 *>(cw + c);
                w[0] = w4.x; w[1] = w4.y; w[2] = w4.z; w[3] = w4.w;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float t0, t1;
                ffma2(t0, t1, __uint_as_float(r[c + 2 * i]), __uint_as_float(r[c + 2 * i + 1]), scale_log2, scale_log2, neg_m, neg_m);
                const float p0 = ex2(t0), p1 = ex2(t1);
                if (FAR) ffma2(ls[2 * i], ls[2 * i + 1], p0, p1, w[2 * i], w[2 * i + 1], ls[2 * i], ls[2 * i + 1]);
                else fadd2(ls[2 * i], ls[2 * i + 1], ls[2 * i], ls[2 * i + 1], p0, p1);
                pk[2 * j + i] = pack16<F16>(p0, p1);
            }
        }
        tmem_st16(p_addr + 16 * half, pk);
        sum += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    }
    return sum;
}

// One row's scores of 64 columns, those of excluded keys set to -inf.  lo, hi: valid columns of the 64 (kDiag, kBdA, kBdB).
__device__ __forceinline__ void t4_scores(uint32_t s_addr, int kind, bool has_empty, int lo, int hi, const float *cw, uint32_t (&r)[64])
{
    tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
    tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
    tc_wait_ld();
    if (kind == kFar) {
        if (has_empty) t4_mask_empty(r, cw);
    } else if (kind != kFull) {
        t4_mask_range(r, lo, hi);
    }
}

}  // namespace vq
