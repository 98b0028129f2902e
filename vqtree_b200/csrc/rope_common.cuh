// Vector loads and the half-split rotation, shared by the kernels that rotate rows (rope.cu, paged_cache.cu).
#pragma once

#include "vq_common.cuh"

namespace vq {

template <typename T> struct RopeVec;
template <> struct RopeVec<float> {
    static constexpr int kN = 4;
    __device__ static void load(const float *p, float (&f)[4])
    {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
    __device__ static void store(float *p, const float (&f)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct RopeVec<__nv_bfloat16> {
    static constexpr int kN = 8;
    __device__ static void load(const __nv_bfloat16 *p, float (&f)[8])
    {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static void store(__nv_bfloat16 *p, const float (&f)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <> struct RopeVec<__half> {
    static constexpr int kN = 8;
    __device__ static void load(const __half *p, float (&f)[8])
    {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = Pair16<__half>::unpack(w[i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
    __device__ static void store(__half *p, const float (&f)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = Pair16<__half>::pack(f[2 * i], f[2 * i + 1]);
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// N table entries; the table rows start on 16-byte boundaries (D/2 and d are multiples of four floats): 128-bit loads
template <int N>
__device__ __forceinline__ void rope_table(const float *t, float (&v)[N])
{
    static_assert(N % 4 == 0, "vector width");
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float4 x = __ldg(reinterpret_cast<const float4 *>(t) + i);
        v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
    }
}
// out = x * cos + rotate_half(x) * sin for the kN elements at d (first half) and d + D/2 (second half)
template <int N>
__device__ __forceinline__ void rope_apply(const float (&x1)[N], const float (&x2)[N], const float (&cv)[N], const float (&sv)[N], float (&o1)[N], float (&o2)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        o1[i] = __fadd_rn(__fmul_rn(x1[i], cv[i]), __fmul_rn(-x2[i], sv[i]));
        o2[i] = __fadd_rn(__fmul_rn(x2[i], cv[i]), __fmul_rn(x1[i], sv[i]));
    }
}
template <int N>
__device__ __forceinline__ void rope_rotate(const float (&x1)[N], const float (&x2)[N], const float *c, const float *s, float (&o1)[N], float (&o2)[N])
{
    float cv[N], sv[N];
    rope_table<N>(c, cv);
    rope_table<N>(s, sv);
    rope_apply<N>(x1, x2, cv, sv, o1, o2);
}

}  // namespace vq
