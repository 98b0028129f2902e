// 8-bit codes of a cache row as 16-bit floats.
#pragma once

#include "vq_common.cuh"

namespace vq {

template <typename T> struct IsBf16 { static constexpr bool value = false; };
template <> struct IsBf16<__nv_bfloat16> { static constexpr bool value = true; };

// Four 8-bit codes -> two packed pairs of 16-bit floats, exactly.
template <typename T> struct Codes8;
template <> struct Codes8<__half> {
    // 0x6400 | (x + 128) is the half 1024 + x + 128
    static __device__ __forceinline__ void expand(uint32_t w, uint32_t &lo, uint32_t &hi)
    {
        w ^= 0x80808080u;
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), bias);
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    }
    // the same times powers of two from 2^-24 to 2^5 (one per place of a pair): exact as well
    static __device__ __forceinline__ void expand_scaled(uint32_t w, __half2 pow2, uint32_t &lo, uint32_t &hi)
    {
        w ^= 0x80808080u;
        const __half2 bias = __hmul2(pow2, __halves2half2(__ushort_as_half(0xe480), __ushort_as_half(0xe480)));   // -1152
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 x = __hfma2(*reinterpret_cast<const __half2 *>(&a), pow2, bias), y = __hfma2(*reinterpret_cast<const __half2 *>(&b), pow2, bias);
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    }
};

// A weight times a value row of codes with scale vs, in halves: weight * (vs * 2^k) and codes * 2^-k, with k such that the first factor lies in
// [1, 2) - and inside what a half holds for every scale of half values (2^-31 .. 2^10).  Otherwise a small scale would put
// the products among the subnormal halves, where the codes of a snapshot (weights without a scale) share the accumulator.
// k goes by the row's own scale: one for several rows would take the bits of the weights of the small ones.
__device__ __forceinline__ int half_weight_shift(float vs)
{
    const int k = 127 - static_cast<int>((__float_as_uint(vs) >> 23) & 255u);
    return min(24, max(-5, k));
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
__device__ __forceinline__ float half_weight_factor(float vs, float &pow2)
{
    const int k = half_weight_shift(vs);
    pow2 = pow2f(-k);
    return vs * pow2f(k);
}

template <> struct Codes8<__nv_bfloat16> {
    // 0x4300 | (x & 127) is the bf16 128 + (x & 127), 0x4300 | (x & 128) is 128 or 256: their difference is x
    static __device__ __forceinline__ uint32_t pair(uint32_t e)
    {
        const uint32_t a = e & 0xff7fff7fu, b = e & 0xff80ff80u;
        const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
        return *reinterpret_cast<const uint32_t *>(&x);
    }
    static __device__ __forceinline__ void expand(uint32_t w, uint32_t &lo, uint32_t &hi)
    {
        lo = pair(__byte_perm(w, 0x43434343u, 0x4140));
        hi = pair(__byte_perm(w, 0x43434343u, 0x4342));
    }
};

}  // namespace vq
