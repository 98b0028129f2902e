// Attention of new tokens over a paged cache: the entry point, and the kernel for fp32.
//
// Row i of a sequence: keys [max(0,i-W), i] scored q1.k1, keys [b, max(0,i-W)) scored q2.k3, everything before the boundary
// b = max(0, (i-W)/128*128) through the counts and value sums per code of that boundary's snapshot - one softmax over all of them.
//
// paged_simt_kernel: one warp per query row.  32 keys at a time: lane l scores key l (its row in 16-byte pieces against the query row in
// shared memory), the warp agrees on a running maximum, then the lanes turn to the D output columns and add 32 weighted value rows.
// fp32 products and sums throughout.
#include "paged_attn.cuh"

namespace vq {

template <typename KV> struct KeyVec;      // 16 bytes of a stored row as fp32
template <> struct KeyVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const float *p, float (&f)[4])
    {
        const float4 v = __ldg(reinterpret_cast<const float4 *>(p));
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
};
template <typename T> struct KeyVec16 {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const T *p, float (&f)[8])
    {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = Pair16<T>::unpack(w[i]);
            f[2 * i] = x.x; f[2 * i + 1] = x.y;
        }
    }
};
template <> struct KeyVec<__nv_bfloat16> : KeyVec16<__nv_bfloat16> {};
template <> struct KeyVec<__half> : KeyVec16<__half> {};
template <> struct KeyVec<int8_t> {
    static constexpr int N = 16;
    static __device__ __forceinline__ void load(const int8_t *p, float (&f)[16])
    {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = static_cast<float>(static_cast<int8_t>(w[i / 4] >> (8 * (i % 4))));
    }
};

template <typename KV, int D>
__device__ __forceinline__ float row_dot(const KV *row, const float *q)
{
    constexpr int N = KeyVec<KV>::N;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int d = 0; d < D; d += N) {
        float f[N];
        KeyVec<KV>::load(row + d, f);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i & 3] = fmaf(f[i], q[d + i], acc[i & 3]);
    }
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

constexpr int kSimtWarps = 8;

template <int D>
struct SimtRow {
    static constexpr int C = D / 32;                     // output columns per lane
    float m = -INFINITY, l = 0.f, o[C];
    __device__ __forceinline__ SimtRow()
    {
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = 0.f;
    }
    // 32 scores (log2 units, -inf: excluded) with denominator weights w and factors f of the value rows; vrow: lane's value row
    template <typename V>
    __device__ __forceinline__ void step(float s, float w, float f, const V *vrow, int lane)
    {
        float mx = s;
#pragma unroll
        for (int x = 16; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, x));
        // A NaN score is no maximum, and as a weight it reaches the sums; with nothing but NaN and excluded keys so far any reference will do
        if (__any_sync(~0u, s != s) && mx == -INFINITY) mx = 0.f;
        if (mx > m) {
            const float a = exp2f(m - mx);
            m = mx;
            l *= a;
#pragma unroll
            for (int c = 0; c < C; ++c) o[c] *= a;
        }
        const bool in = !(s == -INFINITY);
        if (m == -INFINITY) return;                      // warp-uniform: every key so far is excluded
        const float p = in ? exp2f(s - m) : 0.f;
        l += in ? p * w : 0.f;
        const float pf = in ? p * f : 0.f;
        const unsigned some = __ballot_sync(~0u, in);
        for (unsigned left = some; left; left &= left - 1) {
            const int j = __ffs(left) - 1;
            const float pj = __shfl_sync(~0u, pf, j);
            const V *v = reinterpret_cast<const V *>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(vrow), j)) + lane * C;
#pragma unroll
            for (int c = 0; c < C; ++c) o[c] = fmaf(pj, static_cast<float>(v[c]), o[c]);
        }
    }
};

template <typename T, typename KV, int D>
__global__ void __launch_bounds__(kSimtWarps * 32) paged_simt_kernel(const PagedAttnParams p)
{
    constexpr int C = D / 32;
    __shared__ float sq[kSimtWarps][2][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = blockIdx.x * static_cast<int64_t>(kSimtWarps) + warp;
    const int64_t t = item / p.Hq;
    const int hq = static_cast<int>(item - t * p.Hq), hk = hq / p.G;
    if (t >= p.seqs.T) return;
    const int s = p.seqs.find(t);
    int t0, q, n;
    if (s >= p.seqs.S || !p.seqs.seq(s, t0, q, n, p.max_q) || t < t0) return;
    const int i = n - q + static_cast<int>(t - t0), b = p.boundary(i);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        sq[warp][0][lane * C + c] = to_f32(static_cast<const T *>(p.q1)[t * p.q1_t + hq * p.q1_h + lane * C + c]);
        sq[warp][1][lane * C + c] = to_f32(static_cast<const T *>(p.q2)[t * p.q2_t + hq * p.q2_h + lane * C + c]);
    }
    __syncwarp();
    const float *q1 = sq[warp][0], *q2 = p.rerope ? sq[warp][1] : sq[warp][0];
    SimtRow<D> row;
    const int snap = p.snapshot(s, b);
    if (snap >= 0) {
        const T *cb = static_cast<const T *>(p.cb) + static_cast<int64_t>(hk) * p.MK * D;
        const int64_t base = (static_cast<int64_t>(snap) * p.Hkv + hk) * p.MK;
        for (int r0 = 0; r0 < p.MK; r0 += 32) {
            const int r = r0 + lane;
            const float cnt = __ldg(p.cnt + base + r);
            const float sc = cnt > 0.f ? row_dot<T, D>(cb + static_cast<int64_t>(r) * D, sq[warp][1]) * p.scale_log2 : -INFINITY;
            row.step(sc, cnt, 1.f, static_cast<const T *>(p.vsum) + (base + r) * D, lane);
        }
    }
    const int mask = (1 << p.seqs.log_p) - 1;
    for (int j0 = b; j0 <= i; j0 += 32) {
        const int j = j0 + lane;
        float sc = -INFINITY, f = 1.f;
        const KV *vrow = nullptr;
        if (j <= i) {
            const int page = p.seqs.page(s, j >> p.seqs.log_p), r = j & mask;
            if (page >= 0) {
                const bool old = p.rerope && j < i - p.W;
                const PagedPool &kp = old ? p.k3 : p.k1;
                sc = row_dot<KV, D>(static_cast<const KV *>(kp.ptr) + kp.row(page, hk, r), old ? q2 : q1);
                if constexpr (sizeof(KV) == 1) {
                    sc *= __ldg(kp.scale + kp.scale_at(page, hk, r));
                    f = __ldg(p.v.scale + p.v.scale_at(page, hk, r));
                }
                sc *= p.scale_log2;
                vrow = static_cast<const KV *>(p.v.ptr) + p.v.row(page, hk, r);
            }
        }
        row.step(sc, 1.f, f, vrow, lane);
    }
    float l = row.l;
#pragma unroll
    for (int x = 16; x; x >>= 1) l += __shfl_xor_sync(~0u, l, x);
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) static_cast<T *>(p.out)[t * p.o_t + hq * p.o_h + lane * C + c] = from_f32<T>(row.o[c] * inv);
}

template <typename T, typename KV>
static int launch_simt(const PagedAttnParams &p, cudaStream_t stream)
{
    const int64_t rows = p.seqs.T * p.Hq, grid = (rows + kSimtWarps - 1) / kSimtWarps;
    if (grid > 0x7fffffff) return VQ_EUNSUPPORTED;
    if (p.D == 64) paged_simt_kernel<T, KV, 64><<<static_cast<unsigned>(grid), kSimtWarps * 32, 0, stream>>>(p);
    else paged_simt_kernel<T, KV, 128><<<static_cast<unsigned>(grid), kSimtWarps * 32, 0, stream>>>(p);
    return launch_status();
}

template <typename T>
static int launch_simt_kv(const PagedAttnParams &p, bool q8, cudaStream_t stream)
{
    return q8 ? launch_simt<T, int8_t>(p, stream) : launch_simt<T, T>(p, stream);
}

}  // namespace vq

extern "C" int vqattn_paged_attention(const VqPagedAttentionArgs *a, void *stream)
{
    using namespace vq;
    if (a == nullptr) return VQ_EINVAL_ARG;
    int st = check_basic(&a->q1, 3);
    if (st != VQ_OK) return st;
    const int64_t T = a->q1.shape[0], Hq = a->q1.shape[1];
    const int dt = a->q1.dtype;
    if (!is_act_dtype(dt)) return VQ_EINVAL_DTYPE;
    PagedArgs kv;
    if ((st = check_paged_kv(a->kv, T, a->status_word, kv)) != VQ_OK) return st;
    if (kv.dtype != VQ_I8 && kv.dtype != dt) return VQ_EINVAL_DTYPE;
    for (const VqTensorDesc *t : {&a->q1, &a->q2, &a->out})
        if ((st = check_tokens(*t, T, Hq, kv.D, dt)) != VQ_OK) return st;
    if (Hq % kv.Hkv != 0) return VQ_EINVAL_SHAPE;
    if (a->window <= 0 || a->window % kBlock != 0 || a->window > 0x40000000 || a->max_q <= 0) return VQ_EINVAL_ARG;
    const int64_t G = Hq / kv.Hkv;
    if (G > 128) return VQ_EUNSUPPORTED;
    PagedAttnParams p{};
    if (a->codebook.ptr != nullptr) {
        if ((st = check_basic(&a->codebook, 3)) != VQ_OK || (st = check_basic(&a->cnt, 3)) != VQ_OK || (st = check_basic(&a->vsum, 4)) != VQ_OK ||
            (st = check_basic(&a->snap_table, 2)) != VQ_OK)
            return st;
        if (a->codebook.dtype != dt || a->vsum.dtype != dt || a->cnt.dtype != VQ_F32 || a->snap_table.dtype != VQ_I32) return VQ_EINVAL_DTYPE;
        const int64_t MK = a->codebook.shape[1], NS = a->cnt.shape[0];
        if (a->codebook.shape[0] != kv.Hkv || a->codebook.shape[2] != kv.D) return VQ_EINVAL_SHAPE;
        if (a->cnt.shape[1] != kv.Hkv || a->cnt.shape[2] != MK) return VQ_EINVAL_SHAPE;
        if (a->vsum.shape[0] != NS || a->vsum.shape[1] != kv.Hkv || a->vsum.shape[2] != MK || a->vsum.shape[3] != kv.D) return VQ_EINVAL_SHAPE;
        if (a->snap_table.shape[0] != kv.seqs.S) return VQ_EINVAL_SHAPE;
        if (MK % kBlock != 0 || MK > (1 << 24) || NS > 0x7fffffff || a->snap_table.shape[1] > (1 << 24)) return VQ_EUNSUPPORTED;
        if (!is_dense(a->codebook) || !is_dense(a->cnt) || !is_dense(a->vsum)) return VQ_EINVAL_STRIDE;
        for (const VqTensorDesc *t : {&a->codebook, &a->cnt, &a->vsum})
            if (reinterpret_cast<uintptr_t>(t->ptr) % 16) return VQ_EINVAL_STRIDE;
        p.cb = a->codebook.ptr; p.cnt = static_cast<const float *>(a->cnt.ptr); p.vsum = a->vsum.ptr;
        p.snap = static_cast<const int32_t *>(a->snap_table.ptr); p.snap_row = a->snap_table.stride[0];
        p.MS = static_cast<int>(a->snap_table.shape[1]); p.NS = static_cast<int>(NS); p.MK = static_cast<int>(MK);
    }
    const VqTensorDesc *all[] = {&a->q1, &a->q2, &a->out, &a->codebook, &a->cnt, &a->vsum, &a->snap_table};
    if ((st = check_device(all, a->codebook.ptr ? 7 : 3)) != VQ_OK || (st = check_paged_devices(a->kv)) != VQ_OK) return st;
    p.k1 = kv.k1; p.k3 = kv.k3; p.v = kv.v; p.seqs = kv.seqs; p.rerope = kv.rerope;
    p.Hq = static_cast<int>(Hq); p.Hkv = kv.Hkv; p.G = static_cast<int>(G); p.D = kv.D;
    p.q1 = a->q1.ptr; p.q2 = a->q2.ptr; p.out = a->out.ptr;
    p.q1_t = a->q1.stride[0]; p.q1_h = a->q1.stride[1]; p.q2_t = a->q2.stride[0]; p.q2_h = a->q2.stride[1];
    p.o_t = a->out.stride[0]; p.o_h = a->out.stride[1];
    p.W = static_cast<int>(a->window);
    p.max_q = static_cast<int>(a->max_q < T ? a->max_q : T);
    p.scale_log2 = (a->scale > 0.f ? a->scale : 1.0f / sqrtf(static_cast<float>(kv.D))) * 1.4426950408889634f;
    p.wait_limit = wait_limit_cycles();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool q8 = kv.dtype == VQ_I8;
    if (is_16bit(dt) && static_cast<int64_t>(p.max_q) * G <= kFewRows) return launch_paged_few(p, dt, q8, s);
    if (is_16bit(dt)) return launch_paged_chunk(p, dt, q8, s);
    return launch_simt_kv<float>(p, q8, s);
}
