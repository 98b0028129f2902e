// Writing new tokens into the pages of a cache and reading rows back.
//
// Append: every token brings Hkv keys, Hkv values and Hq queries.  A group of lanes owns one to four of these rows - each lane 16 bytes of the
// first half and the matching 16 of the second, so a rotation needs no exchange - and finds the token's sequence by bisecting cu_q
// (every lane of a token reads the same words).  8-bit rows: scale = max|x| * (1/127), code = rint(x * (1/scale)); the maximum is an
// exchange inside the group, x is the fp32 rotation (quantising a rotation already rounded to 16 bits would round twice), and every
// operation is rounded on its own, so codes and scales are reproducible bit for bit.  Division-free per element: one reciprocal a row.
// Read: a thread per 16 bytes of stored rows.  Both are bound by memory traffic, and by their launch when there are few rows.
#include "paged_common.cuh"
#include "rope_common.cuh"

#include <type_traits>

namespace vq {

__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// rint(x * inv) of four values, as bytes.  Adding 1.5 * 2^23 rounds to the nearest even integer and leaves it in the low bits (|x * inv| is at
// most 127 and a few units): two additions of the fp32 pipe instead of a conversion of the slower one.
__device__ __forceinline__ uint32_t four_codes(float x0, float x1, float x2, float x3, float inv)
{
    constexpr float kMagic = 12582912.f;
    const uint32_t b0 = __float_as_uint(__fadd_rn(__fmul_rn(x0, inv), kMagic)), b1 = __float_as_uint(__fadd_rn(__fmul_rn(x1, inv), kMagic));
    const uint32_t b2 = __float_as_uint(__fadd_rn(__fmul_rn(x2, inv), kMagic)), b3 = __float_as_uint(__fadd_rn(__fmul_rn(x3, inv), kMagic));
    return __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
}

// One row, N elements of the first half in a and N of the second in b, written to a pool in its own type or as 8-bit codes with a scale.
// g_mask: the lanes that share the row.
template <typename T, typename KV, int D>
struct RowStore {
    static constexpr int N = RopeVec<T>::kN, LPR = D / 2 / N;
    static __device__ __forceinline__ void put(const PagedPool &pool, int page, int head, int r, int l, unsigned g_mask, const float (&a)[N],
                                               const float (&b)[N])
    {
        KV *dst = static_cast<KV *>(const_cast<void *>(pool.ptr)) + pool.row(page, head, r) + l * N;
        if constexpr (sizeof(KV) == 1) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) m = max_nan(m, max_nan(fabsf(a[i]), fabsf(b[i])));
#pragma unroll
            for (int o = LPR / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(g_mask, m, o));
            float scale = __fmul_rn(m, 1.0f / 127.0f);
            if (scale < 1.17549435e-38f) scale = 0.f;
            const bool finite = scale < INFINITY;                    // false for NaN too
            const float inv = finite && scale > 0.f ? __frcp_rn(scale) : 0.f;
            uint32_t lo[N / 4], hi[N / 4];
#pragma unroll
            for (int w = 0; w < N / 4; ++w) {
                lo[w] = four_codes(a[4 * w], a[4 * w + 1], a[4 * w + 2], a[4 * w + 3], inv);
                hi[w] = four_codes(b[4 * w], b[4 * w + 1], b[4 * w + 2], b[4 * w + 3], inv);
            }
            if (!finite) {
#pragma unroll
                for (int w = 0; w < N / 4; ++w) lo[w] = hi[w] = 0;
            }
            if constexpr (N == 8) {
                *reinterpret_cast<uint2 *>(dst) = make_uint2(lo[0], lo[1]);
                *reinterpret_cast<uint2 *>(dst + D / 2) = make_uint2(hi[0], hi[1]);
            } else {
                *reinterpret_cast<uint32_t *>(dst) = lo[0];
                *reinterpret_cast<uint32_t *>(dst + D / 2) = hi[0];
            }
            if (l == 0) const_cast<float *>(pool.scale)[pool.scale_at(page, head, r)] = finite ? scale : __int_as_float(0x7fffffff);
        } else {
            RopeVec<KV>::store(dst, a);
            RopeVec<KV>::store(dst + D / 2, b);
        }
    }
};

struct AppendParams {
    PagedPool k1, k3, v;
    PagedSeqs seqs;
    bool raw;                    // raw keys of their own
    int Hkv, Hq;                 // Hq 0: no queries
    const void *k, *vin, *q;
    void *q1, *q2;
    int64_t k_t, k_h, v_t, v_h, q_t, q_h, q1_t, q1_h, q2_t, q2_h;   // strides in elements
    const float *cos_tab, *sin_tab;
    int64_t n_pos, const_pos;
    uint32_t items;              // groups of heads of all tokens
};

// A group of lanes takes U heads of one kind - keys, values or queries - of a token: they share the look-ups and the table's row, which is twice a
// 16-bit row.  Three CTAs of an SM leave 80 registers a thread: four heads of 16 bits on their way to 8 spill 344 bytes there (stored; 908 loaded).
template <typename T, typename KV, int D, int U>
__global__ void __launch_bounds__(256, sizeof(KV) == 1 ? 3 : 2) paged_append_kernel(const AppendParams p)
{
    using St = RowStore<T, KV, D>;
    constexpr int N = St::N, LPR = St::LPR;
    const int l = threadIdx.x % LPR;
    const uint32_t item = blockIdx.x * (256u / LPR) + threadIdx.x / LPR;
    if (item >= p.items) return;                                     // whole groups leave together
    const unsigned g_mask = (LPR == 32 ? 0xffffffffu : (1u << LPR) - 1u) << (threadIdx.x % 32 / LPR * LPR);
    const uint32_t kg = (p.Hkv + U - 1) / U, per = 2 * kg + (p.Hq + U - 1) / U, t = item / per, r = item - t * per;
    const bool is_q = r >= 2 * kg, is_v = !is_q && r >= kg;
    const int h0 = static_cast<int>(is_q ? r - 2 * kg : is_v ? r - kg : r) * U, heads = min(U, (is_q ? p.Hq : p.Hkv) - h0);
    const int64_t sh = is_q ? p.q_h : is_v ? p.v_h : p.k_h;
    const T *src = (is_q ? static_cast<const T *>(p.q) + t * p.q_t : is_v ? static_cast<const T *>(p.vin) + t * p.v_t
                                                                        : static_cast<const T *>(p.k) + t * p.k_t) + h0 * sh + l * N;
    float x1[U][N], x2[U][N], o1[N], o2[N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const T *row = src + (u < heads ? u : 0) * sh;
        RopeVec<T>::load(row, x1[u]);
        RopeVec<T>::load(row + D / 2, x2[u]);
    }
    const int s = p.seqs.find(t);
    if (s >= p.seqs.S) return;                                       // behind the last sequence
    int t0, q, n;
    if (!p.seqs.seq(s, t0, q, n) || t < static_cast<uint32_t>(t0)) return;
    const int pos = n - q + (static_cast<int>(t) - t0), pr = pos & ((1 << p.seqs.log_p) - 1);
    int page = 0;
    if (!is_q) {
        page = p.seqs.page(s, pos >> p.seqs.log_p);
        if (page < 0) return;
    }
    if (is_v) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u < heads) St::put(p.v, page, h0 + u, pr, l, g_mask, x1[u], x2[u]);
        return;
    }
    const bool turn = p.cos_tab != nullptr;
    float cv[N], sv[N];
    if (turn) {
        int64_t at = pos;
        if (at >= p.n_pos) {
            at = p.n_pos - 1;
            p.seqs.raise(VQ_WORD_BAD_POSITION);
        }
        rope_table<N>(p.cos_tab + at * (D / 2) + l * N, cv);
        rope_table<N>(p.sin_tab + at * (D / 2) + l * N, sv);
    }
    auto rotate = [&](int u) {
        if (turn) {
            rope_apply<N>(x1[u], x2[u], cv, sv, o1, o2);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            o1[i] = x1[u][i];
            o2[i] = x2[u][i];
        }
    };
    if (!is_q) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= heads) continue;
            rotate(u);
            St::put(p.k1, page, h0 + u, pr, l, g_mask, o1, o2);
            if (p.raw) St::put(p.k3, page, h0 + u, pr, l, g_mask, x1[u], x2[u]);
        }
        return;
    }
    auto queries = [&](void *out, int64_t st, int64_t shd) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= heads) continue;
            rotate(u);
            T *dst = static_cast<T *>(out) + t * st + (h0 + u) * shd + l * N;
            RopeVec<T>::store(dst, o1);
            RopeVec<T>::store(dst + D / 2, o2);
        }
    };
    queries(p.q1, p.q1_t, p.q1_h);
    if (p.q2 == nullptr) return;
    if (turn) {
        rope_table<N>(p.cos_tab + p.const_pos * (D / 2) + l * N, cv);
        rope_table<N>(p.sin_tab + p.const_pos * (D / 2) + l * N, sv);
    }
    queries(p.q2, p.q2_t, p.q2_h);
}

// byte j of w, which is code + 128, as the code's fp32 value: 2^23 + w[j] - (2^23 + 128)
__device__ __forceinline__ float code_f32(uint32_t w, int j) { return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | j)) - 8388736.f; }

struct ReadParams {
    PagedPool pool[3];
    void *out[3];
    const int32_t *table, *start, *lens;
    int64_t t_row;
    int MB, NP, log_p, S, Hkv, n;
    uint64_t items;              // 16-byte pieces of one pool's rows
    int32_t *status;
};

// A thread takes 16 bytes of U rows, whose loads are under way together.  Eight CTAs of an SM: the way to a row is a chain of loads (length, table,
// row), which only more threads can hide.
template <typename KV, typename O, int D, int U>
__global__ void __launch_bounds__(256, 8) paged_read_kernel(const ReadParams p)
{
    constexpr int N = 16 / sizeof(KV), LPR = D / N, STEP = 256 / LPR;
    const int which = blockIdx.y, l = threadIdx.x % LPR;
    const uint64_t row0 = blockIdx.x * static_cast<uint64_t>(U * STEP) + threadIdx.x / LPR, rows = p.items / LPR;
    if (row0 >= rows) return;
    uint32_t s, h, r;
    if (rows <= 0xffffffffu) {                                       // the usual case: divisions in 32 bits
        const uint32_t w = static_cast<uint32_t>(row0), sh = w / p.n;
        r = w - sh * p.n;
        s = sh / p.Hkv;
        h = sh - s * p.Hkv;
    } else {
        const uint64_t sh = row0 / p.n;
        r = static_cast<uint32_t>(row0 - sh * p.n);
        s = static_cast<uint32_t>(sh / p.Hkv);
        h = static_cast<uint32_t>(sh - static_cast<uint64_t>(s) * p.Hkv);
    }
    const PagedPool &pool = p.pool[which];
    uint4 in[U];
    float scale[U];
    bool there[U];
    const KV *head = static_cast<const KV *>(pool.ptr) + h * pool.s_head + l * N;
    const float *head_scale = pool.scale + h * pool.c_head;
    int start = __ldg(p.start + s), len = __ldg(p.lens + s);
    const int32_t *table = p.table + s * p.t_row;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        there[u] = false;
        in[u] = make_uint4(0, 0, 0, 0);
        scale[u] = 0.f;
        if (row0 + u * STEP < rows) {
            const int64_t pos = static_cast<int64_t>(start) + r;
            if (pos >= 0 && pos < len) {
                const int col = static_cast<int>(pos) >> p.log_p, pr = static_cast<int>(pos) & ((1 << p.log_p) - 1);
                const int page = col < p.MB ? __ldg(table + col) : -1;
                if (page < 0 || page >= p.NP) {
                    if (p.status) atomicExch(p.status, VQ_WORD_BAD_PAGE);
                } else {
                    there[u] = true;
                    in[u] = *reinterpret_cast<const uint4 *>(head + page * pool.s_page + pr * pool.s_row);
                    if constexpr (sizeof(KV) == 1) scale[u] = __ldg(head_scale + page * pool.c_page + pr * pool.c_row);
                }
            }
        }
        if (u + 1 == U || row0 + (u + 1) * STEP >= rows) continue;
        r += STEP;
        if (r < static_cast<uint32_t>(p.n)) continue;
        do {
            r -= p.n;
            if (++h == static_cast<uint32_t>(p.Hkv)) {
                h = 0;
                ++s;
            }
        } while (r >= static_cast<uint32_t>(p.n));
        head = static_cast<const KV *>(pool.ptr) + h * pool.s_head + l * N;
        head_scale = pool.scale + h * pool.c_head;
        start = __ldg(p.start + s);
        len = __ldg(p.lens + s);
        table = p.table + s * p.t_row;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (row0 + u * STEP >= rows) return;
        O *dst = static_cast<O *>(p.out[which]) + (row0 + u * STEP) * D + l * N;
        if constexpr (sizeof(KV) == 1) {
            constexpr int V = RopeVec<O>::kN;
            const uint32_t w[4] = {in[u].x, in[u].y, in[u].z, in[u].w};
#pragma unroll
            for (int i = 0; i < N; i += V) {
                float x[V];
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = there[u] ? __fmul_rn(code_f32(w[(i + j) / 4] ^ 0x80808080u, (i + j) % 4), scale[u]) : 0.f;
                RopeVec<O>::store(dst + i, x);
            }
        } else {
            *reinterpret_cast<uint4 *>(dst) = in[u];
        }
    }
}

// Rows per thread: several where there are many CTAs anyway, one where there are few.  Measured with several / with one, us: appending 2048 tokens
// of 32 kv heads, 16 bits 29.8 / 32.5; second turns of 12 sequences, 8 bits, with reading them back 120 / 132; reading 16 windows of 2303 rows,
// 32 heads, 8 bits to half (915 MB) 162 / 215.
constexpr int kManyCtas = 148 * 8;      // eight for each SM of the chip

template <typename T, typename KV, int D>
static int launch_append(AppendParams &p, cudaStream_t stream)
{
    constexpr int U = 4;
    constexpr uint32_t per = 256u / RowStore<T, KV, D>::LPR;
    const int64_t T_ = p.seqs.T;
    const bool many = T_ * (2 * p.Hkv + p.Hq) / per >= static_cast<int64_t>(U) * kManyCtas;
    const int u = many ? U : 1;
    p.items = static_cast<uint32_t>(T_ * (2 * ((p.Hkv + u - 1) / u) + (p.Hq + u - 1) / u));
    const uint32_t grid = (p.items + per - 1) / per;
    if (many) paged_append_kernel<T, KV, D, U><<<grid, 256, 0, stream>>>(p);
    else paged_append_kernel<T, KV, D, 1><<<grid, 256, 0, stream>>>(p);
    return launch_status();
}

template <typename T, typename KV>
static int launch_append(AppendParams &p, int D, cudaStream_t stream)
{
    return D == 64 ? launch_append<T, KV, 64>(p, stream) : launch_append<T, KV, 128>(p, stream);
}

template <typename KV, typename O, int D>
static int launch_read(ReadParams &p, int pools, cudaStream_t stream)
{
    constexpr int U = 2;
    p.items = static_cast<uint64_t>(p.S) * p.Hkv * p.n * (D * sizeof(KV) / 16);
    const uint64_t blocks = (p.items + 255) / 256;
    if (blocks > 0x7fffffffu) return VQ_EUNSUPPORTED;
    if (blocks * pools >= U * kManyCtas)
        paged_read_kernel<KV, O, D, U><<<dim3(static_cast<unsigned>((blocks + U - 1) / U), static_cast<unsigned>(pools)), 256, 0, stream>>>(p);
    else
        paged_read_kernel<KV, O, D, 1><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(pools)), 256, 0, stream>>>(p);
    return launch_status();
}

template <typename KV, typename O>
static int launch_read(ReadParams &p, int D, int pools, cudaStream_t stream)
{
    return D == 64 ? launch_read<KV, O, 64>(p, pools, stream) : launch_read<KV, O, 128>(p, pools, stream);
}

}  // namespace vq

extern "C" int vqattn_paged_append(const VqPagedAppendArgs *a, void *stream)
{
    using namespace vq;
    if (a == nullptr) return VQ_EINVAL_ARG;
    int st = check_basic(&a->k, 3);
    if (st != VQ_OK) return st;
    const int64_t T = a->k.shape[0];
    const int dt = a->k.dtype;
    if (!is_act_dtype(dt)) return VQ_EINVAL_DTYPE;
    PagedArgs kv;
    if ((st = check_paged_kv(a->kv, T, a->status_word, kv)) != VQ_OK) return st;
    if (kv.dtype != VQ_I8 && kv.dtype != dt) return VQ_EINVAL_DTYPE;
    // several writers of one row, of one scale, of one query
    const auto same = [](const VqTensorDesc &x, const VqTensorDesc &y) { return x.ptr != nullptr && x.ptr == y.ptr; };
    const VqPagedKv &pg = a->kv;
    if (same(pg.k3, pg.k1) || same(pg.v, pg.k1) || same(pg.v, pg.k3)) return VQ_EINVAL_ARG;
    if (same(pg.k3_scale, pg.k1_scale) || same(pg.v_scale, pg.k1_scale) || same(pg.v_scale, pg.k3_scale) || same(a->q1, a->q2)) return VQ_EINVAL_ARG;
    if ((st = check_tokens(a->k, T, kv.Hkv, kv.D, dt)) != VQ_OK) return st;
    if ((st = check_tokens(a->v, T, kv.Hkv, kv.D, dt)) != VQ_OK) return st;
    const bool has_q = a->q.ptr != nullptr;
    const int64_t Hq = has_q ? a->q.shape[1] : 0;
    if (has_q) {
        if ((st = check_tokens(a->q, T, Hq, kv.D, dt)) != VQ_OK) return st;
        if ((st = check_tokens(a->q1, T, Hq, kv.D, dt)) != VQ_OK) return st;
        if (a->q2.ptr != nullptr && (st = check_tokens(a->q2, T, Hq, kv.D, dt)) != VQ_OK) return st;
    }
    for (const VqTensorDesc *t : {&a->kv.k1, &a->kv.k3, &a->kv.v, &a->kv.k1_scale, &a->kv.k3_scale, &a->kv.v_scale, &a->q1, &a->q2})
        if (expanded(*t)) return VQ_EINVAL_STRIDE;
    if ((a->cos_tab == nullptr) != (a->sin_tab == nullptr)) return VQ_EINVAL_ARG;
    if (a->cos_tab != nullptr) {
        if (a->n_pos <= 0 || (has_q && a->q2.ptr != nullptr && (a->const_pos < 0 || a->const_pos >= a->n_pos))) return VQ_EINVAL_ARG;
        if (reinterpret_cast<uintptr_t>(a->cos_tab) % 16 || reinterpret_cast<uintptr_t>(a->sin_tab) % 16) return VQ_EINVAL_STRIDE;
    }
    const int64_t rows = 2 * kv.Hkv + Hq;
    if (T * rows > 0x7fffffffLL) return VQ_EUNSUPPORTED;
    const VqTensorDesc *all[] = {&a->k, &a->v, has_q ? &a->q : nullptr, has_q ? &a->q1 : nullptr, has_q ? &a->q2 : nullptr};
    if ((st = check_device(all, 5)) != VQ_OK || (st = check_paged_devices(a->kv)) != VQ_OK) return st;
    AppendParams p{};
    p.k1 = kv.k1; p.k3 = kv.k3; p.v = kv.v; p.seqs = kv.seqs; p.raw = kv.rerope;
    p.Hkv = kv.Hkv; p.Hq = static_cast<int>(Hq);
    p.k = a->k.ptr; p.vin = a->v.ptr; p.q = a->q.ptr; p.q1 = a->q1.ptr; p.q2 = a->q2.ptr;
    p.k_t = a->k.stride[0]; p.k_h = a->k.stride[1]; p.v_t = a->v.stride[0]; p.v_h = a->v.stride[1];
    p.q_t = a->q.stride[0]; p.q_h = a->q.stride[1]; p.q1_t = a->q1.stride[0]; p.q1_h = a->q1.stride[1];
    p.q2_t = a->q2.stride[0]; p.q2_h = a->q2.stride[1];
    p.cos_tab = a->cos_tab; p.sin_tab = a->sin_tab; p.n_pos = a->n_pos; p.const_pos = a->const_pos;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kv.dtype == VQ_I8) {
        if (dt == VQ_F32) return launch_append<float, int8_t>(p, kv.D, s);
        return dt == VQ_F16 ? launch_append<__half, int8_t>(p, kv.D, s) : launch_append<__nv_bfloat16, int8_t>(p, kv.D, s);
    }
    if (dt == VQ_F32) return launch_append<float, float>(p, kv.D, s);
    return dt == VQ_F16 ? launch_append<__half, __half>(p, kv.D, s) : launch_append<__nv_bfloat16, __nv_bfloat16>(p, kv.D, s);
}

extern "C" int vqattn_paged_read(const VqPagedReadArgs *a, void *stream)
{
    using namespace vq;
    if (a == nullptr || a->pool[0].ptr == nullptr) return VQ_EINVAL_ARG;
    ReadParams p{};
    int64_t shape[4] = {0, 0, 0, 0};
    int st = check_basic(&a->pool[0], 4);
    if (st != VQ_OK) return st;
    const int dt = a->pool[0].dtype, odt = a->out[0].dtype;
    if (!is_pool_dtype(dt) || !is_act_dtype(odt) || (dt != VQ_I8 && odt != dt)) return VQ_EINVAL_DTYPE;
    int pools = 0;
    const VqTensorDesc *all[12];
    int na = 0;
    for (; pools < 3 && a->pool[pools].ptr != nullptr; ++pools) {
        if ((st = check_pool(a->pool[pools], a->scale[pools], shape, dt, p.pool[pools])) != VQ_OK) return st;
        const VqTensorDesc &o = a->out[pools];
        if ((st = check_basic(&o, 4)) != VQ_OK) return st;
        if (o.dtype != odt) return VQ_EINVAL_DTYPE;
        for (int i = 0; i < 4; ++i)
            if (o.shape[i] != (i == 1 ? shape[1] : i == 3 ? shape[3] : a->out[0].shape[i])) return VQ_EINVAL_SHAPE;
        if (!is_dense(o) || reinterpret_cast<uintptr_t>(o.ptr) % 16) return VQ_EINVAL_STRIDE;
        p.out[pools] = o.ptr;
        all[na++] = &a->pool[pools]; all[na++] = &a->scale[pools]; all[na++] = &o;
    }
    if (shape[3] != 64 && shape[3] != 128) return VQ_EUNSUPPORTED;
    if (log2_page(shape[2]) < 0) return VQ_EUNSUPPORTED;
    if (shape[0] > 0x7fffffff || shape[1] > 65535) return VQ_EUNSUPPORTED;
    if ((st = check_basic(&a->table, 2)) != VQ_OK) return st;
    if (a->table.dtype != VQ_I32) return VQ_EINVAL_DTYPE;
    const int64_t S = a->table.shape[0], n = a->out[0].shape[2];
    if (a->out[0].shape[0] != S) return VQ_EINVAL_SHAPE;
    if (S > (1 << 20) || a->table.shape[1] > (1 << 24) || n > 0x7fffffff) return VQ_EUNSUPPORTED;
    if ((st = check_i32(a->start, S)) != VQ_OK || (st = check_i32(a->lens, S)) != VQ_OK) return st;
    all[na++] = &a->table; all[na++] = &a->start; all[na++] = &a->lens;
    if ((st = check_device(all, na)) != VQ_OK) return st;
    p.table = static_cast<const int32_t *>(a->table.ptr); p.t_row = a->table.stride[0];
    p.start = static_cast<const int32_t *>(a->start.ptr); p.lens = static_cast<const int32_t *>(a->lens.ptr);
    p.MB = static_cast<int>(a->table.shape[1]); p.NP = static_cast<int>(shape[0]); p.log_p = log2_page(shape[2]);
    p.S = static_cast<int>(S); p.Hkv = static_cast<int>(shape[1]); p.n = static_cast<int>(n);
    p.status = a->status_word;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int D = static_cast<int>(shape[3]);
    if (dt == VQ_I8) {
        if (odt == VQ_F32) return launch_read<int8_t, float>(p, D, pools, s);
        return odt == VQ_F16 ? launch_read<int8_t, __half>(p, D, pools, s) : launch_read<int8_t, __nv_bfloat16>(p, D, pools, s);
    }
    if (dt == VQ_F32) return launch_read<float, float>(p, D, pools, s);
    return dt == VQ_F16 ? launch_read<__half, __half>(p, D, pools, s) : launch_read<__nv_bfloat16, __nv_bfloat16>(p, D, pools, s);
}
