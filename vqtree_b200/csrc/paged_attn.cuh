// Parameters of the attention over a paged cache and what its kernels share.
#pragma once

#include "paged_common.cuh"

namespace vq {

struct PagedAttnParams {
    PagedPool k1, k3, v;
    PagedSeqs seqs;
    bool rerope;                 // keys before the exact window are scored q2.k3
    int Hq, Hkv, G, D;
    const void *q1, *q2;
    void *out;
    int64_t q1_t, q1_h, q2_t, q2_h, o_t, o_h;      // strides in elements
    const void *cb, *vsum;       // [Hkv,MK,D], [NS,Hkv,MK,D]; cb NULL: local part only
    const float *cnt;            // [NS,Hkv,MK]
    const int32_t *snap;         // [S,MS]
    int64_t snap_row;
    int MS, NS, MK;
    int W;                       // window
    int max_q;
    float scale_log2;            // softmax scale * log2(e)
    long long wait_limit;

    __device__ __forceinline__ int boundary(int i) const { return i > W ? (i - W) / kBlock * kBlock : 0; }
    // snapshot of boundary b of sequence s; -1: none is wanted, or the table names none (reported)
    __device__ __forceinline__ int snapshot(int s, int b) const { return checked_snapshot(b, snapshot_entry(s, b)); }
    // the same in two parts: what the table says, and the check
    __device__ __forceinline__ int snapshot_entry(int s, int b) const
    {
        return b > 0 && cb != nullptr ? __ldg(snap + s * snap_row + (b / kBlock) % MS) : -1;
    }
    __device__ __forceinline__ int checked_snapshot(int b, int id) const
    {
        if (b <= 0 || cb == nullptr) return -1;
        if (id >= 0 && id < NS) return id;
        seqs.raise(VQ_WORD_BAD_PAGE);
        return -1;
    }
};

constexpr int kFewRows = 32;     // query rows (tokens times query heads of a kv head) of the few-token kernel
int launch_paged_few(const PagedAttnParams &p, int dtype, bool q8, cudaStream_t stream);
int launch_paged_chunk(const PagedAttnParams &p, int dtype, bool q8, cudaStream_t stream);

}  // namespace vq
