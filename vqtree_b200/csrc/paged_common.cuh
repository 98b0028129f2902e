// Shared by the kernels of the paged cache: what a token's row is, where a key lies, argument checks.
#pragma once

#include "vq_common.cuh"

namespace vq {

// One pool of rows [NP,Hkv,P,D], strides in elements; scales (8-bit rows) [NP,Hkv,P].
struct PagedPool {
    const void *ptr;
    int64_t s_page, s_head, s_row;
    const float *scale;
    int64_t c_page, c_head, c_row;
    __device__ __forceinline__ int64_t row(int page, int head, int r) const { return page * s_page + head * s_head + r * s_row; }
    __device__ __forceinline__ int64_t scale_at(int page, int head, int r) const { return page * c_page + head * c_head + r * c_row; }
};

// Sequences: page table, packed new tokens, lengths.
struct PagedSeqs {
    const int32_t *table;
    int64_t t_row;               // elements between the rows of the table
    int MB, NP, log_p;           // columns, pages in the pool, log2 of the page size
    const int32_t *cu_q, *lens;
    int S;
    int64_t T;                   // rows of the packed tensors
    int32_t *status;

    __device__ __forceinline__ void raise(int word) const
    {
        if (status) atomicExch(status, word);
    }
    // page of token block `col` of sequence s, -1 (and the status word) when there is none
    __device__ __forceinline__ int page(int s, int col) const
    {
        const int pg = col >= 0 && col < MB ? __ldg(table + s * t_row + col) : -1;
        if (pg >= 0 && pg < NP) return pg;
        raise(VQ_WORD_BAD_PAGE);
        return -1;
    }
    // New tokens [t0, t0 + q) of sequence s, the last of n tokens.  False: the lengths do not fit.
    __device__ __forceinline__ bool seq(int s, int &t0, int &q, int &n, int64_t max_q = 0x7fffffff) const
    {
        t0 = __ldg(cu_q + s);
        q = __ldg(cu_q + s + 1) - t0;
        n = __ldg(lens + s);
        if (q == 0) return true;
        if (t0 >= 0 && q > 0 && t0 + static_cast<int64_t>(q) <= T && q <= n && q <= max_q && n <= static_cast<int64_t>(MB) << log_p) return true;
        raise(VQ_WORD_BAD_LENGTH);
        return false;
    }
    // Sequence of packed row t (cu_q does not decrease), S when it belongs to none.
    __device__ __forceinline__ int find(int64_t t) const
    {
        int lo = 0, hi = S;      // first s with cu_q[s + 1] > t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (__ldg(cu_q + mid + 1) > t) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    }
};

// code * scale of an 8-bit row, rounded to fp32
__device__ __forceinline__ float dequant(int8_t c, float scale) { return __fmul_rn(static_cast<float>(c), scale); }

// ------------------------------------------------------------------------------------------ host side

inline bool is_pool_dtype(int dt) { return is_act_dtype(dt) || dt == VQ_I8; }
inline int dtype_size(int dt) { return dt == VQ_I8 ? 1 : dt == VQ_F32 ? 4 : 2; }

// rows that start on 16 bytes: base and every outer stride
inline bool rows_aligned(const VqTensorDesc &t)
{
    const int64_t v = 16 / dtype_size(t.dtype);
    for (int i = 0; i + 1 < t.ndim; ++i)
        if (t.shape[i] > 1 && (t.stride[i] % v != 0 || t.stride[i] < 0)) return false;
    return reinterpret_cast<uintptr_t>(t.ptr) % 16 == 0;
}

// an expanded tensor: several elements in one place
inline bool expanded(const VqTensorDesc &t)
{
    if (t.ptr == nullptr) return false;
    for (int i = 0; i < t.ndim; ++i)
        if (t.shape[i] > 1 && t.stride[i] == 0) return true;
    return false;
}

// int32 vector of n entries, contiguous
inline int check_i32(const VqTensorDesc &t, int64_t n)
{
    int st = check_basic(&t, 1);
    if (st != VQ_OK) return st;
    if (t.dtype != VQ_I32) return VQ_EINVAL_DTYPE;
    return t.shape[0] == n ? VQ_OK : VQ_EINVAL_SHAPE;
}

// A pool against the expected shape (np <= 0: any; then *np is set) and type.
inline int check_pool(const VqTensorDesc &t, const VqTensorDesc &scale, int64_t shape[4], int dtype, PagedPool &out)
{
    int st = check_basic(&t, 4);
    if (st != VQ_OK) return st;
    if (t.dtype != dtype) return VQ_EINVAL_DTYPE;
    for (int i = 0; i < 4; ++i) {
        if (shape[i] <= 0) shape[i] = t.shape[i];
        if (t.shape[i] != shape[i]) return VQ_EINVAL_SHAPE;
    }
    if (!rows_aligned(t)) return VQ_EINVAL_STRIDE;
    out = PagedPool{t.ptr, t.stride[0], t.stride[1], t.stride[2], nullptr, 0, 0, 0};
    if ((dtype == VQ_I8) != (scale.ptr != nullptr)) return VQ_EINVAL_ARG;
    if (dtype == VQ_I8) {
        if (scale.ndim != 3) return VQ_EINVAL_SHAPE;
        if (scale.dtype != VQ_F32) return VQ_EINVAL_DTYPE;
        for (int i = 0; i < 3; ++i) {
            if (scale.shape[i] != shape[i]) return VQ_EINVAL_SHAPE;
            if (scale.stride[i] < 0) return VQ_EINVAL_STRIDE;
        }
        if (reinterpret_cast<uintptr_t>(scale.ptr) % 4) return VQ_EINVAL_STRIDE;
        out.scale = static_cast<const float *>(scale.ptr);
        out.c_page = scale.stride[0]; out.c_head = scale.stride[1]; out.c_row = scale.stride[2];
    }
    return VQ_OK;
}

inline int log2_page(int64_t P) { return P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : -1; }

struct PagedArgs {
    PagedPool k1, k3, v;
    PagedSeqs seqs;
    bool rerope;                 // raw keys of their own
    int Hkv, D, P, dtype;
};

// Everything of a VqPagedKv but the device (the caller checks it with its own tensors).  T: rows of the packed tensors.
inline int check_paged_kv(const VqPagedKv &kv, int64_t T, int32_t *status, PagedArgs &p)
{
    int64_t shape[4] = {0, 0, 0, 0};
    const int dt = kv.k1.dtype;
    if (kv.k1.ptr == nullptr) return VQ_EINVAL_ARG;
    if (!is_pool_dtype(dt)) return VQ_EINVAL_DTYPE;
    int st = check_pool(kv.k1, kv.k1_scale, shape, dt, p.k1);
    if (st != VQ_OK) return st;
    if ((st = check_pool(kv.v, kv.v_scale, shape, dt, p.v)) != VQ_OK) return st;
    p.rerope = kv.k3.ptr != nullptr;
    if (p.rerope) {
        if ((st = check_pool(kv.k3, kv.k3_scale, shape, dt, p.k3)) != VQ_OK) return st;
    } else {
        p.k3 = p.k1;
    }
    if (shape[3] != 64 && shape[3] != 128) return VQ_EUNSUPPORTED;
    if (log2_page(shape[2]) < 0) return VQ_EUNSUPPORTED;
    if (shape[0] > 0x7fffffff || shape[1] > 65535) return VQ_EUNSUPPORTED;
    if ((st = check_basic(&kv.table, 2)) != VQ_OK) return st;
    if (kv.table.dtype != VQ_I32) return VQ_EINVAL_DTYPE;
    const int64_t S = kv.table.shape[0];
    if (S > (1 << 20) || kv.table.shape[1] > (1 << 30) / shape[2] || T > 0x7fffffff) return VQ_EUNSUPPORTED;   // positions stay below 2^30
    if ((st = check_i32(kv.cu_q, S + 1)) != VQ_OK) return st;
    if ((st = check_i32(kv.lens, S)) != VQ_OK) return st;
    p.seqs = PagedSeqs{static_cast<const int32_t *>(kv.table.ptr), kv.table.stride[0], static_cast<int>(kv.table.shape[1]),
                       static_cast<int>(shape[0]), log2_page(shape[2]), static_cast<const int32_t *>(kv.cu_q.ptr),
                       static_cast<const int32_t *>(kv.lens.ptr), static_cast<int>(S), T, status};
    p.Hkv = static_cast<int>(shape[1]); p.P = static_cast<int>(shape[2]); p.D = static_cast<int>(shape[3]); p.dtype = dt;
    return VQ_OK;
}

inline int check_paged_devices(const VqPagedKv &kv)
{
    const VqTensorDesc *all[] = {&kv.k1, &kv.k3, &kv.v, &kv.k1_scale, &kv.k3_scale, &kv.v_scale, &kv.table, &kv.cu_q, &kv.lens};
    return check_device(all, 9);
}

// packed rows [T,H,D] of one type
inline int check_tokens(const VqTensorDesc &t, int64_t T, int64_t H, int64_t D, int dtype)
{
    int st = check_basic(&t, 3);
    if (st != VQ_OK) return st;
    if (t.dtype != dtype) return VQ_EINVAL_DTYPE;
    if (t.shape[0] != T || t.shape[1] != H || t.shape[2] != D) return VQ_EINVAL_SHAPE;
    return rows_aligned(t) ? VQ_OK : VQ_EINVAL_STRIDE;
}

}  // namespace vq
