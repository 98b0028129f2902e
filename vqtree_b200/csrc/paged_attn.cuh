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
    // 8-bit rows: their blocks as 16-bit floats, [k1, v, k3][ws_blocks][Hkv][128][D], and behind them a factor per row; NULL: none
    void *ws;
    int64_t ws_blocks;

    __device__ __forceinline__ int boundary(int i) const { return i > W ? (i - W) / kBlock * kBlock : 0; }
    __device__ __forceinline__ float *ws_scales(int64_t row_bytes) const { return reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + row_bytes); }
    // first key block that the query at position i sees one by one
    __device__ __forceinline__ int first_block(int i) const { return max(0, i / kBlock - W / kBlock); }
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

// Tokens [pos0, pos0 + ntok) of sequence s (of length n), rows t0 .. of the packed tensors: all in one 128-block of positions, so that they share a
// boundary and its snapshot.
struct ChunkTile {
    int s, t0, ntok, pos0, n, snap;
    int ws0;                     // workspace block of the sequence's key block 0 (may be negative: early blocks are not there)
};

// Tile number -> sequence and tokens, by one warp.  False: there are fewer tiles.
__device__ __forceinline__ bool chunk_find(const PagedAttnParams &p, int TQ, int tile, ChunkTile &out)
{
    const int lane = threadIdx.x & 31, per = (kBlock + TQ - 1) / TQ;
    int before = 0, ws_before = 0;
    for (int base = 0; base < p.seqs.S; base += 32) {
        int t0 = 0, q = 0, n = 0, cnt = 0, blocks = 0;
        if (base + lane < p.seqs.S && p.seqs.seq(base + lane, t0, q, n, p.max_q) && q > 0) {
            const int i0 = n - q, nb = (n - 1) / kBlock - i0 / kBlock + 1;
            cnt = nb == 1 ? (q + TQ - 1) / TQ
                          : (kBlock - i0 % kBlock + TQ - 1) / TQ + (nb - 2) * per + ((n - 1) % kBlock + TQ) / TQ;
            blocks = (n - 1) / kBlock - p.first_block(i0) + 1;
        }
        int sum = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += x;
        }
        int ws_sum = blocks;
        if (p.ws != nullptr) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(~0u, ws_sum, o);
                if (lane >= o) ws_sum += x;
            }
        }
        const unsigned mine = __ballot_sync(~0u, before + sum > tile);
        if (mine) {
            const int l = __ffs(mine) - 1;
            int x = tile - before - (__shfl_sync(~0u, sum, l) - __shfl_sync(~0u, cnt, l));   // tile of the sequence
            t0 = __shfl_sync(~0u, t0, l);
            q = __shfl_sync(~0u, q, l);
            n = __shfl_sync(~0u, n, l);
            int i0 = n - q;
            const int head = (min(kBlock - i0 % kBlock, q) + TQ - 1) / TQ;                   // tiles of its first block
            int blk = i0 / kBlock;
            if (x >= head) {
                x -= head;
                blk += 1 + x / per;
                x %= per;
            }
            const int lo = max(i0, blk * kBlock) + x * TQ, hi = min(min(n, (blk + 1) * kBlock), lo + TQ);
            out.s = base + l;
            out.t0 = t0 + lo - i0;
            out.ntok = hi - lo;
            out.pos0 = lo;
            out.n = n;
            out.snap = p.snapshot(out.s, p.boundary(lo));
            const int ws_end = ws_before + __shfl_sync(~0u, ws_sum, l);
            out.ws0 = ws_end - __shfl_sync(~0u, blocks, l) - p.first_block(i0);
            if (p.ws != nullptr && ws_end > p.ws_blocks) {       // only where sequences share rows (cu_q decreases in between): their blocks may be
                p.seqs.raise(VQ_WORD_BAD_LENGTH);                // more than the workspace was sized for
                return false;
            }
            return true;
        }
        before += __shfl_sync(~0u, sum, 31);
        ws_before += __shfl_sync(~0u, ws_sum, 31);
    }
    return false;
}

// An upper bound of the number of tiles, known without the lengths: every block that a sequence touches rounds its tokens up.
inline int64_t chunk_tiles(const PagedSeqs &q, int TQ)
{
    const int64_t tiles = q.T / TQ + q.T / kBlock + 2 * static_cast<int64_t>(q.S);
    return tiles < q.T ? tiles : q.T;
}

// Blocks of 128 keys that the new tokens of a call can see, at most.
inline int64_t paged_blocks(int64_t S, int64_t T, int64_t window) { return S * (window / kBlock + 3) + T / kBlock; }
// 8-bit rows: converting a block once per call pays where its keys meet several query tiles.  Measured, us, first / on the way, 32 query heads over 8,
// D = 128, MK1024, window 2048 (512), new tokens per sequence: 2 tiles each, 8 sequences 131 / 160 (80 / 83); 4 tiles, 8 sequences 176 / 238 (109 /
// 122), 24 sequences 414 / 561 (255 / 291); 16 tiles, 2 sequences 118 / 166 (77 / 88).  The line is at four: below it the workspace grows
// faster than what it saves.  It goes by the average, known without the lengths: a long chunk among many single tokens is converted on the way.
inline bool convert_first(int64_t S, int64_t T, int64_t G) { return T * G >= 4 * kBlock * S; }

constexpr int kFewRows = 32;     // query rows (tokens times query heads of a kv head) of the few-token kernel
int launch_paged_few(const PagedAttnParams &p, int dtype, bool q8, cudaStream_t stream);
int launch_paged_f32(const PagedAttnParams &p, bool q8, cudaStream_t stream);
int launch_paged_chunk(const PagedAttnParams &p, int dtype, bool q8, cudaStream_t stream);

}  // namespace vq
