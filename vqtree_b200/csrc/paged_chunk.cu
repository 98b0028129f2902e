// Attention over a paged cache for chunks of new tokens, on the sm_100a tensor cores.
//
// One CTA owns up to 128 query rows of one kv head - its G query heads times 128 / G tokens of one sequence, all in one 128-block of positions,
// so that they share a boundary and every tile of keys and values is fetched once for all heads of the group - and walks their
// work items with one online softmax: codebook tiles against the boundary's snapshot, the boundary block (raw keys, then rotated ones), the
// blocks between, the causal block.  The softmax protocol is that of the prefill kernel with 128-key steps (prefill_tc4.cu): score buffers in
// tensor memory that P overwrites, one thread per row and buffer, a reference maximum handed from step to step, lazily raised.
// Which rows a tile has is read on the device (one warp counts the tiles of 32 sequences at a time), so a captured call may be
// replayed with other lengths.
//   16-bit rows   a thread loads pages by TMA, 128 / P boxes a tile, into a ring of four 32 KB slots.
//   8-bit rows    where a call's sequences bring four query tiles each, on the average, and the caller gave a workspace, a kernel before this one turns
//                 every block's codes into 16-bit floats (exact) there once, with a factor per row beside them, and this one loads tiles of it as above.
//                 Otherwise codes arrive by TMA in two staging tiles and three warps convert them into a ring of three slots, in the swizzled layout
//                 the tensor cores read.  The scales of a step's keys multiply scores, those of its values weights, per column.
// Bound by the hand-offs between the softmax warps and the tensor pipe, as the prefill kernel is.  Measured: 4096 tokens at
// context 32768, 32 heads, D = 128, MK1024, W1024, bf16: 252 us, 560 TFLOP/s.  Six second turns of 700 tokens and fewer, 32 query heads over 8, 8-bit rows:
// 203 us, 20 of them converting (converted on the way 283, by plain loads one tile ahead 410; 16-bit rows 162).
// The softmax over 8-bit rows spills 112 - 188 bytes a thread (128 registers; scores, factors of keys and of values).
// Weights are rounded to 16 bits before they meet their values, as in the prefill kernels: P is an operand of the tensor pipe.  Their sum is not.
// Rows behind a sequence's end hold anything: their scores are masked and their value rows are zeroed before the product.
#include "codes8.cuh"
#include "paged_attn.cuh"
#include "tc_softmax.cuh"

#include <type_traits>

namespace vq {

constexpr int kChunkPages = 256;        // page table entries of a tile kept in shared memory; the rest is read where it is needed

// CONV: 8-bit rows converted on their way into the ring
template <int D, bool CONV>
struct ChunkCfg {
    static constexpr int kBufs = 3;                           // S/P buffers = softmax warpgroups
    static constexpr int kSoft = 4 * kBufs;                   // softmax warps
    static constexpr int kLoad = CONV ? 3 : 1;                  // loading warps: 16 warps of 128 registers with 8-bit rows
    static constexpr int kWarpMma = kSoft, kWarpLoad = kSoft + 1;
    static constexpr int kThreads = (kSoft + 1 + kLoad) * 32;
    static constexpr int NH = D / 64;
    static constexpr int kTile = NH * kHalfBytes;             // 128 x D
    static constexpr int kSlots = CONV ? 3 : 4;
    static constexpr int kRaw = kBlock * D;                   // 128 rows of codes
    static constexpr int kQ = 0, kRing = 2 * kTile, kRaws = kRing + kSlots * kTile;
    static constexpr int kTotal = kRaws + (CONV ? 2 * kRaw : 0) + 1024;   // + slack for 1024-byte alignment
    static constexpr uint32_t kColS = 0, kColO = kBlock * kBufs, kCols = 512;
    static constexpr int kOq = D / 2;
};

struct ChunkParams {
    PagedAttnParams a;
    int TQ;                      // tokens per tile
};

// The tile's items, in order: codebook tiles, boundary block (ReRoPE: two masked passes), blocks between, causal block.
struct ChunkWork {
    int kb0, n_far, n_bd, first_full, n_full, n_items, rerope;
    __device__ __forceinline__ ChunkWork(const PagedAttnParams &p, const ChunkTile &t)
    {
        const int m = t.pos0 / kBlock;
        rerope = p.rerope;
        kb0 = m - p.W / kBlock;
        n_far = t.snap >= 0 ? p.MK / kBlock : 0;
        n_bd = kb0 >= 0 ? (rerope ? 2 : 1) : 0;
        first_full = kb0 >= 0 ? kb0 + 1 : 0;
        n_full = m - first_full;
        n_items = n_far + n_bd + n_full + 1;
    }
    __device__ __forceinline__ int kind(int it) const
    {
        if (it < n_far) return kFar;
        it -= n_far;
        if (it < n_bd) return rerope ? (it == 0 ? kBdA : kBdB) : kFull;
        return it - n_bd < n_full ? kFull : kDiag;
    }
    __device__ __forceinline__ int block(int it) const
    {
        if (it < n_far) return it;
        it -= n_far;
        return it < n_bd ? kb0 : first_full + it - n_bd;
    }
};

__device__ __forceinline__ void fmul2(float &d0, float &d1, float a0, float a1, float b0, float b1)
{
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

// Barrier ID of THREADS threads that tells whether the condition holds in all of them.
template <int ID, int THREADS>
__device__ __forceinline__ bool all_of_named(bool x)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(static_cast<uint32_t>(x)), "n"(ID), "n"(THREADS) : "memory");
    return r != 0;
}

// 8-bit rows.  ks: scale of each of 64 keys times the softmax scale, vs: factor of each value row.
__device__ __forceinline__ void load_scores(uint32_t s_addr, uint32_t (&r)[64])
{
    tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
    tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
    tc_wait_ld();
}
// the largest score, in log2 units; [lo, hi): the columns that count
template <bool MASKED>
__device__ __forceinline__ float q8_max(const uint32_t (&r)[64], int lo, int hi, const float *ks)
{
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 64; c += 4) {
        const float4 k = *reinterpret_cast<const float4 *>(ks + c);
        float x[4];
        fmul2(x[0], x[1], __uint_as_float(r[c]), __uint_as_float(r[c + 1]), k.x, k.y);
        fmul2(x[2], x[3], __uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]), k.z, k.w);
        if (MASKED) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < lo || c + i >= hi) x[i] = -INFINITY;
        }
        mx[(c >> 2) & 3] = fmax3(mx[(c >> 2) & 3], x[0], x[1]);
        mx[((c >> 2) + 1) & 3] = fmax3(mx[((c >> 2) + 1) & 3], x[2], x[3]);
    }
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
// weights times value factors, packed 16-bit floats; returns sum plus the weights.  What does not count weighs nothing, whatever its value is.
template <bool F16, bool MASKED>
__device__ __forceinline__ float q8_exp(const uint32_t (&r)[64], uint32_t p_addr, int lo, int hi, const float *ks, const float *vs, float neg_m, float sum)
{
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float ls[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = 32 * half + 4 * j;
            const float4 k4 = *reinterpret_cast<const float4 *>(ks + c), v4 = *reinterpret_cast<const float4 *>(vs + c);
            const float k[4] = {k4.x, k4.y, k4.z, k4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float t0, t1, w0, w1;
                ffma2(t0, t1, __uint_as_float(r[c + 2 * i]), __uint_as_float(r[c + 2 * i + 1]), k[2 * i], k[2 * i + 1], neg_m, neg_m);
                float p0 = ex2(t0), p1 = ex2(t1);
                const bool out0 = MASKED && (c + 2 * i < lo || c + 2 * i >= hi), out1 = MASKED && (c + 2 * i + 1 < lo || c + 2 * i + 1 >= hi);
                if (out0) p0 = 0.f;
                if (out1) p1 = 0.f;
                fadd2(ls[2 * i], ls[2 * i + 1], ls[2 * i], ls[2 * i + 1], p0, p1);
                fmul2(w0, w1, p0, p1, v[2 * i], v[2 * i + 1]);
                if (out0) w0 = 0.f;
                if (out1) w1 = 0.f;
                pk[2 * j + i] = pack16<F16>(w0, w1);
            }
        }
        tmem_st16(p_addr + 16 * half, pk);
        sum += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    }
    return sum;
}

// SRC: where local rows come from
enum ChunkSrc : int { kPages16 = 0, kPages8 = 1, kWorkspace = 2 };

template <int D, bool F16, int SRC>
__global__ void __launch_bounds__(ChunkCfg<D, SRC == kPages8>::kThreads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap tm_q1, const __grid_constant__ CUtensorMap tm_q2, const __grid_constant__ CUtensorMap tm_k1,
                   const __grid_constant__ CUtensorMap tm_k3, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_cb,
                   const __grid_constant__ CUtensorMap tm_vs, const ChunkParams cp)
{
    constexpr bool Q8 = SRC != kPages16, CONV = SRC == kPages8;
    using C = ChunkCfg<D, CONV>;
    using T = typename std::conditional<F16, __half, __nv_bfloat16>::type;
    constexpr int NH = C::NH, NS = C::kSlots, NB = C::kBufs, kSoftThreads = C::kSoft * 32;
    const PagedAttnParams &p = cp.a;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-ptx::smem_u32(smem_raw) & 1023u);   // stays an address of shared memory for the compiler
    __shared__ __align__(8) uint64_t bar_q, kv_full[NS], kv_empty[NS], s_full[NB], p_full[NB], pv_done[NB], refbar[NB][4], endbar, raw_full[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_err, s_some;
    __shared__ ChunkTile s_tile;
    __shared__ int s_page[kChunkPages];
    __shared__ __align__(16) float s_cw[C::kSoft][kBlock];   // [softmax warp][column]: counts of the codebook tile it works on
    __shared__ float s_ref[kBlock];
    __shared__ float s_lend[NB][kBlock], s_mend[NB][kBlock];
    __shared__ __align__(16) float s_cv[Q8 ? C::kSoft : 1][Q8 ? kBlock : 4];   // 8-bit rows: factors of its weights (s_cw: of its scores)

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hk = blockIdx.y;
    if (warp == 0) {
        ChunkTile t;
        const bool some = chunk_find(p, cp.TQ, blockIdx.x, t);
        if (lane == 0) {
            s_some = some;
            s_tile = t;
        }
    }
    if (tid == C::kWarpMma * 32) {
        mbar_init(&bar_q, 1);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        for (int i = 0; i < NB; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
            for (int g = 0; g < 4; ++g) mbar_init(&refbar[i][g], 1);
        }
        mbar_init(&raw_full[0], 1);
        mbar_init(&raw_full[1], 1);
        mbar_init(&endbar, C::kSoft);
        fence_mbar_init();
        s_err = 0;
    }
    if (tid < kBlock) s_ref[tid] = -INFINITY;
    __syncthreads();
    if (!s_some) return;
    const ChunkTile tile = s_tile;
    const ChunkWork work(p, tile);
    const int n = work.n_items;
    const int n_q2 = p.rerope ? work.n_far + (work.n_bd == 2 ? 1 : 0) : work.n_far;   // items scored with q2 come first
    const int log_p = p.seqs.log_p, col0 = max(work.kb0, 0) * kBlock >> log_p, page_size = 1 << log_p;
    if (warp == C::kWarpMma && elect_one()) {
        prefetch_tmap(&tm_q1); prefetch_tmap(&tm_q2); prefetch_tmap(&tm_cb); prefetch_tmap(&tm_vs);
        mbar_expect_tx(&bar_q, (n_q2 > 0 ? 2 : 1) * NH * 128 * cp.TQ * p.G);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            tma_load_3d(smem + C::kQ + h * kHalfBytes, &tm_q1, &bar_q, 64 * h, hk * p.G, tile.t0);
            if (n_q2 > 0) tma_load_3d(smem + C::kQ + C::kTile + h * kHalfBytes, &tm_q2, &bar_q, 64 * h, hk * p.G, tile.t0);
        }
    }
    {
        const int last = min(tile.n - 1, (tile.pos0 / kBlock + 1) * kBlock - 1) >> log_p;   // page of the last key that is read
        if (tid < kSoftThreads)
            for (int x = tid; x < min(last - col0 + 1, kChunkPages); x += kSoftThreads) s_page[x] = p.seqs.page(tile.s, col0 + x);
    }
    if (warp == C::kWarpLoad) {
        __syncwarp();
        tmem_alloc(&s_tmem, C::kCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    auto page_of = [&](int key) {
        const int x = (key >> log_p) - col0;
        return x < kChunkPages ? s_page[x] : p.seqs.page(tile.s, x + col0);
    };

    if (warp >= C::kWarpLoad) {
        // ================================================================== loads, in the order the tensor pipe consumes them: K0 K1 K2 V0 K3 V1 ...
        const int lw = warp - C::kWarpLoad;
        int slot = 0;
        uint32_t free_par = 1u;
        bool first_round = true, ok = true;
        auto advance = [&]() {
            if (++slot == NS) {
                slot = 0;
                free_par ^= 1u;
                first_round = false;
            }
        };
        auto wait_slot = [&]() { return first_round || mbar_wait(&kv_empty[slot], free_par, p.wait_limit); };
        auto far_tile = [&](int it, bool is_v) {
            uint8_t *dst = smem + C::kRing + slot * C::kTile;
            mbar_expect_tx(&kv_full[slot], C::kTile);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                if (is_v) tma_load_3d(dst + h * kHalfBytes, &tm_vs, &kv_full[slot], 64 * h, work.block(it) * kBlock, tile.snap * p.Hkv + hk);
                else tma_load_3d(dst + h * kHalfBytes, &tm_cb, &kv_full[slot], 64 * h, work.block(it) * kBlock, hk);
            }
        };
        // Lane x has page x of an item's block; -1 for missing ones (reported) and those behind the end, which are not loaded.
        auto page_of_lane = [&](int it) {
            const int key = work.block(it) * kBlock + lane * page_size;
            return lane * page_size < kBlock && key < tile.n ? page_of(key) : -1;
        };
        // their boxes, by one elected thread: put(page, number of the page in the block)
        auto each_page = [&](int mine, auto put) {
            for (unsigned left = __ballot_sync(~0u, mine >= 0); left; left &= left - 1) {
                const int x = __ffs(left) - 1, pg = __shfl_sync(~0u, mine, x);
                if (elect_one()) put(pg, x);
                __syncwarp();
            }
        };
        if constexpr (!CONV) {
            auto load = [&](int it, bool is_v) {
                if (!ok) return;
                const int kind = work.kind(it), mine = kind == kFar || SRC == kWorkspace ? -1 : page_of_lane(it);   // known before the slot is free
                const int bytes = __popc(__ballot_sync(~0u, mine >= 0)) * page_size * D * 2;
                if (!__all_sync(~0u, wait_slot())) {
                    ok = false;
                    return;
                }
                if (kind == kFar) {
                    if (elect_one()) far_tile(it, is_v);
                    __syncwarp();
                } else {
                    const CUtensorMap *tm = is_v ? &tm_v : (kind == kBdA ? &tm_k3 : &tm_k1);
                    uint8_t *dst = smem + C::kRing + slot * C::kTile;
                    if (SRC == kWorkspace) {
                        if (elect_one()) {
                            const int z = (tile.ws0 + work.block(it)) * p.Hkv + hk;
                            mbar_expect_tx(&kv_full[slot], C::kTile);
#pragma unroll
                            for (int h = 0; h < NH; ++h) tma_load_3d(dst + h * kHalfBytes, tm, &kv_full[slot], 64 * h, 0, z);
                        }
                        __syncwarp();
                        advance();
                        return;
                    }
                    if (elect_one()) mbar_expect_tx(&kv_full[slot], bytes);
                    __syncwarp();
                    each_page(mine, [&](int pg, int x) {
#pragma unroll
                        for (int h = 0; h < NH; ++h)
                            tma_load_4d(dst + h * kHalfBytes + x * page_size * 128, tm, &kv_full[slot], 64 * h, 0, hk, pg);
                    });
                }
                advance();
            };
            for (int j = 0; j < NB && j < n; ++j) load(j, false);
            for (int j = 0; j < n; ++j) {
                load(j, true);
                if (j + NB < n) load(j + NB, false);
            }
            if (!ok) s_err = 1;
        } else {
            // CH lanes share a row, 8 codes each: what eight of them write together lies in different banks.  A warp takes every third block of
            // eight rows.
            constexpr int CH = D / 8, RPI = 32 / CH, NI = 8 / RPI;
            const int ch = lane % CH, rsub = lane / CH;
            uint32_t from[NI], to[NI];                                     // offsets inside a block of eight rows, staged and swizzled
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = RPI * i + rsub;
                from[i] = r * D + 8 * ch;
                to[i] = (ch >> 3) * kHalfBytes + r * 128 + (((ch & 7) ^ r) << 4);   // 16-byte piece j of row r lies at j ^ (r % 8)
            }
            // load number -> item and kind of tile
            auto item_of = [&](int x, bool &is_v) {
                const int lead = min(NB, n);
                is_v = false;
                if (x < lead) return x;
                const int y = x - lead;                                    // V0 K(NB) V1 K(NB+1) ... until the keys run out
                if (y < 2 * (n - lead)) {
                    is_v = (y & 1) == 0;
                    return is_v ? y / 2 : lead + y / 2;
                }
                is_v = true;
                return y - (n - lead);
            };
            // the next local load that has not been asked for yet, into staging tile `next_raw % 2` (the first loading warp)
            int ask = 0, next_raw = 0;
            auto stage = [&]() {
                bool is_v = false;
                int it = 0;
                for (; ask < 2 * n; ++ask) {
                    it = item_of(ask, is_v);
                    if (work.kind(it) != kFar) break;
                }
                if (ask == 2 * n) return;
                const int mine = page_of_lane(it), bytes = __popc(__ballot_sync(~0u, mine >= 0)) * page_size * D;
                const CUtensorMap *tm = is_v ? &tm_v : (work.kind(it) == kBdA ? &tm_k3 : &tm_k1);
                uint64_t *bar = &raw_full[next_raw & 1];
                uint8_t *dst = smem + C::kRaws + (next_raw & 1) * C::kRaw;
                if (elect_one()) mbar_expect_tx(bar, bytes);
                __syncwarp();
                each_page(mine, [&](int pg, int x) { tma_load_4d(dst + x * page_size * D, tm, bar, 0, 0, hk, pg); });
                ++ask;
                ++next_raw;
            };
            if (lw == 0) {
                stage();
                stage();
            }
            // Half values: a row's codes are multiplied by a power of two that goes with its scale (the softmax warps put its inverse into the
            // weights).  The scales are asked for one tile of values ahead.  A lane has those of four rows: of the NI that a lane converts in block x / RPI as
            // its row x % RPI, for x = the lane's number (and 32 more, with heads of 64).
            float vsc[4];
            auto value_scales = [&](int x) {
                if constexpr (F16) {
                    bool is_v;
                    if (x >= 2 * n) return;
                    const int it = item_of(x, is_v);
                    if (!is_v || work.kind(it) == kFar) return;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int x4 = lane + 32 * (i / NI), key = work.block(it) * kBlock + x4 / RPI * 8 + RPI * (i % NI) + x4 % RPI;
                        const int pg = key < tile.n ? page_of(key) : -1;
                        vsc[i] = pg >= 0 ? __ldg(p.v.scale + p.v.scale_at(pg, hk, key & (page_size - 1))) : 0.f;
                    }
                }
            };
            auto next_value_scales = [&](int x) {                          // behind values in load x
                bool is_v;
                item_of(x + 1, is_v);
                value_scales(is_v ? x + 1 : x + 2);
            };
            int raw = 0;
            value_scales(min(NB, n));
            for (int x = 0; x < 2 * n; ++x) {
                bool is_v;
                const int it = item_of(x, is_v);
                const bool far = work.kind(it) == kFar;
                ok = wait_slot() && (far || mbar_wait(&raw_full[raw & 1], (raw >> 1) & 1, p.wait_limit));
                ok = all_of_named<2, C::kLoad * 32>(ok);                   // the loading warps leave together or not at all
                if (!ok) break;
                if (far) {
                    if (lw == 0 && elect_one()) far_tile(it, is_v);
                    __syncwarp();
                    if (is_v) next_value_scales(x);
                } else {
                    const uint8_t *src = smem + C::kRaws + (raw & 1) * C::kRaw;
                    uint8_t *dst = smem + C::kRing + slot * C::kTile;
                    uint32_t p2s[2];                                       // of those rows, two halves a word
                    if (F16 && is_v) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            p2s[i] = ptx::pack_f16(pow2f(-half_weight_shift(vsc[2 * i])), pow2f(-half_weight_shift(vsc[2 * i + 1])));
                        next_value_scales(x);
                    }
                    auto convert = [&](auto scaled) {
#pragma unroll 1
                        for (int blk = lw; blk < kBlock / 8; blk += C::kLoad) {
                            uint2 codes[NI];
                            uint32_t p2_of[2] = {0, 0};
                            if constexpr (scaled.value) {
                                p2_of[0] = __shfl_sync(~0u, NI == 4 || blk < 8 ? p2s[0] : p2s[1], (blk * RPI + rsub) & 31);
                                if (NI == 4) p2_of[1] = __shfl_sync(~0u, p2s[1], (blk * RPI + rsub) & 31);
                            }
#pragma unroll
                            for (int i = 0; i < NI; ++i) codes[i] = *reinterpret_cast<const uint2 *>(src + blk * (8 * D) + from[i]);
#pragma unroll
                            for (int i = 0; i < NI; ++i) {
                                uint4 w;
                                if constexpr (scaled.value) {
                                    const uint32_t h = __byte_perm(p2_of[i / 2], 0, i & 1 ? 0x3232 : 0x1010);
                                    const __half2 p2 = *reinterpret_cast<const __half2 *>(&h);
                                    Codes8<__half>::expand_scaled(codes[i].x, p2, w.x, w.y);
                                    Codes8<__half>::expand_scaled(codes[i].y, p2, w.z, w.w);
                                } else {
                                    Codes8<T>::expand(codes[i].x, w.x, w.y);
                                    Codes8<T>::expand(codes[i].y, w.z, w.w);
                                }
                                *reinterpret_cast<uint4 *>(dst + blk * 1024 + to[i]) = w;
                            }
                        }
                    };
                    if constexpr (F16) {
                        if (is_v) convert(std::true_type());
                        else convert(std::false_type());
                    } else {
                        convert(std::false_type());
                    }
                    fence_proxy_async_smem();
                    asm volatile("bar.sync 1, %0;" ::"n"(C::kLoad * 32) : "memory");   // staging tile read, slot written
                    if (lw == 0) {
                        if (elect_one()) mbar_arrive(&kv_full[slot]);
                        __syncwarp();
                        stage();
                    }
                    ++raw;
                }
                advance();
            }
            if (!ok) s_err = 1;
        }
    } else if (warp == C::kWarpMma) {
        // ================================================================== products
        if (elect_one()) {
            constexpr uint32_t idesc_qk = idesc_f16kind(128, kBlock, 0, 0, F16 ? 0u : 1u);
            constexpr uint32_t idesc_pv = idesc_f16kind(128, D, 0, 1, F16 ? 0u : 1u);
            const uint64_t d_q = smem_desc_sw128(smem_u32(smem + C::kQ), 16, 1024);
            const uint64_t d_k0 = smem_desc_sw128(smem_u32(smem + C::kRing), 16, 1024);
            const uint64_t d_v0 = smem_desc_sw128(smem_u32(smem + C::kRing), kHalfBytes, 1024);
            bool ok = mbar_wait(&bar_q, 0, p.wait_limit);
            int slot = 0;
            uint32_t slot_par = 0;
            int sbuf = 0, pbuf = 0;
            uint32_t p_par = 0;
            auto next_slot = [&]() {
                if (++slot == NS) {
                    slot = 0;
                    slot_par ^= 1u;
                }
            };
            auto qk = [&](int it) {
                if (!ok) return;
                if (!mbar_wait(&kv_full[slot], slot_par, p.wait_limit)) {
                    ok = false;
                    return;
                }
                tc_fence_after();
                const uint64_t db = d_k0 + static_cast<uint64_t>((slot * C::kTile) >> 4);
                const uint64_t da = d_q + static_cast<uint64_t>((it < n_q2 ? C::kTile : 0) >> 4);
                const uint32_t sdst = tmem + C::kColS + kBlock * sbuf;
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int k4 = 0; k4 < 4; ++k4) {
                        const uint64_t off = static_cast<uint64_t>((h * kHalfBytes + k4 * 32) >> 4);
                        if (h == 0 && k4 == 0) mma_ss_first(sdst, da + off, db + off, idesc_qk);
                        else mma_ss_acc(sdst, da + off, db + off, idesc_qk);
                    }
                tc_commit(&kv_empty[slot]);
                tc_commit(&s_full[sbuf]);
                next_slot();
                if (++sbuf == NB) sbuf = 0;
            };
            auto pv = [&](int it) {
                if (!ok) return;
                if (!mbar_wait(&p_full[pbuf], p_par, p.wait_limit) || !mbar_wait(&kv_full[slot], slot_par, p.wait_limit)) {
                    ok = false;
                    return;
                }
                tc_fence_after();
                const uint64_t dv = d_v0 + static_cast<uint64_t>((slot * C::kTile) >> 4);
                const uint32_t odst = tmem + C::kColO, psrc = tmem + C::kColS + kBlock * pbuf;
                if (it == 0) mma_ts_first(odst, psrc, dv, idesc_pv);
                else mma_ts_acc(odst, psrc, dv, idesc_pv);
#pragma unroll
                for (int kk = 1; kk < kBlock / 16; ++kk) mma_ts_acc(odst, psrc + 8 * kk, dv + static_cast<uint64_t>((kk * 2048) >> 4), idesc_pv);
                tc_commit(&kv_empty[slot]);
                tc_commit(&pv_done[pbuf]);
                next_slot();
                if (++pbuf == NB) {
                    pbuf = 0;
                    p_par ^= 1u;
                }
            };
            for (int j = 0; j < NB && j < n; ++j) qk(j);
            for (int j = 0; j < n; ++j) {
                pv(j);
                if (j + NB < n) qk(j + NB);
            }
            if (!ok) s_err = 1;
        }
    } else {
        // ================================================================== softmax
        constexpr unsigned kAll = 0xffffffffu;
        const int g = warp >> 2, lq = warp & 3;
        const int row = lq * 32 + lane;
        const int rpos = tile.pos0 % kBlock + row / p.G;      // position of the row's token inside its block (rows without a token: behind it)
        const uint32_t lane_off = static_cast<uint32_t>(lq * 32) << 16;
        const uint32_t sa = tmem + lane_off + C::kColS + kBlock * g;
        const uint32_t o_addr = tmem + lane_off + C::kColO;
        float my_ref = -INFINITY, l_part = 0.f;
        bool ok = true;
        constexpr int NCW = kBlock / 32;
        const float *cnt_base = p.cnt + (static_cast<int64_t>(max(tile.snap, 0)) * p.Hkv + hk) * p.MK + lane;
        float *cw = &s_cw[warp][0], *cv = &s_cv[Q8 ? warp : 0][0];
        // Lane l fetches what goes with columns l, 32 + l, ... of one of the warp's steps ahead: counts of codes; scales of 8-bit keys and values.
        float reg_w[NCW], reg_v[Q8 ? NCW : 1];
        auto ahead = [&](int it) {
            if (it < work.n_far) {
#pragma unroll
                for (int i = 0; i < NCW; ++i) reg_w[i] = __ldg(cnt_base + it * kBlock + 32 * i);
            } else if constexpr (SRC == kWorkspace) {
                if (it >= n) return;
                const float *f = p.ws_scales(3 * p.ws_blocks * p.Hkv * (kBlock * D * 2)) + (static_cast<int64_t>(tile.ws0 + work.block(it)) * p.Hkv + hk) * kBlock + lane;
                const int64_t pool = p.ws_blocks * p.Hkv * kBlock, from = work.kind(it) == kBdA ? 2 * pool : 0;
#pragma unroll
                for (int i = 0; i < NCW; ++i) {
                    reg_w[i] = __ldg(f + from + 32 * i);
                    reg_v[i] = __ldg(f + pool + 32 * i);
                }
            } else if constexpr (Q8) {
                if (it >= n) return;
                const bool old = work.kind(it) == kBdA;
                const float *ks = old ? p.k3.scale : p.k1.scale;
                const int64_t c_page = old ? p.k3.c_page : p.k1.c_page, c_head = old ? p.k3.c_head : p.k1.c_head, c_row = old ? p.k3.c_row : p.k1.c_row;
#pragma unroll
                for (int i = 0; i < NCW; ++i) {
                    const int key = work.block(it) * kBlock + 32 * i + lane, pg = key < tile.n ? page_of(key) : -1, r = key & (page_size - 1);
                    reg_w[i] = pg >= 0 ? __ldg(ks + pg * c_page + hk * c_head + r * c_row) : 0.f;
                    reg_v[i] = pg >= 0 ? __ldg(p.v.scale + p.v.scale_at(pg, hk, r)) : 0.f;
                }
            }
        };
        ahead(g);
#pragma unroll 1
        for (int it = g; it < n; it += NB) {
            const int par = (it / NB) & 1;
            const int kind = work.kind(it);
            const bool q8 = Q8 && kind != kFar;
            bool has_empty = false;
            if (kind == kFar || q8) {
                __syncwarp();
                bool full = true;
#pragma unroll
                for (int i = 0; i < NCW; ++i) {
                    if (kind == kFar) {
                        cw[32 * i + lane] = reg_w[i];
                        full = full && reg_w[i] > 0.f;
                    } else if constexpr (Q8) {
                        cw[32 * i + lane] = CONV ? reg_w[i] * p.scale_log2 : reg_w[i];
                        float p2;
                        cv[32 * i + lane] = CONV && F16 ? half_weight_factor(reg_v[i], p2) : reg_v[i];
                    }
                }
                has_empty = kind == kFar && __any_sync(kAll, !full);
                __syncwarp();
                ahead(it + NB);
            }
            const int lo = kind == kBdB ? rpos : 0, hi = kind == kDiag ? rpos + 1 : kind == kBdA ? rpos : kBlock;
            if (!__all_sync(kAll, mbar_wait(&s_full[g], par, p.wait_limit))) {
                ok = false;
                break;
            }
            tc_fence_after();
            uint32_t r[64];
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < kBlock; c += 64) {
                if (Q8 && q8) {
                    load_scores(sa + c, r);
                    mx = fmaxf(mx, kind == kFull ? q8_max<false>(r, 0, 64, cw + c) : q8_max<true>(r, lo - c, hi - c, cw + c));
                } else {
                    t4_scores(sa + c, kind, has_empty, lo - c, hi - c, cw + c, r);
                    mx = fmaxf(mx, t4_max(r));
                }
            }
            const float m_tile = q8 ? mx : mx * p.scale_log2;
            if (it > 0 && !__all_sync(kAll, mbar_wait(&refbar[(g + NB - 1) % NB][lq], ((it - 1) / NB) & 1, p.wait_limit))) {
                ok = false;
                break;
            }
            const float ref = s_ref[row];
            float m_use = ref;
            if (m_tile > ref + kT4Lazy || ref == -INFINITY) m_use = fmaxf(ref, m_tile);
            if (m_use != ref) s_ref[row] = m_use;
            __syncwarp();
            if (lane == 0) mbar_arrive(&refbar[g][lq]);
            const float m_safe = (m_use == -INFINITY) ? 0.f : m_use;
            const bool rescale = (m_use != ref) && (ref != -INFINITY);
            if (__any_sync(kAll, rescale)) {
                if (!__all_sync(kAll, mbar_wait(&pv_done[(it - 1) % NB], ((it - 1) / NB) & 1, p.wait_limit))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const float alpha = rescale ? ex2(ref - m_safe) : 1.f;
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16(o_addr + 16 * c, o);
                    tc_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                    tmem_st16(o_addr + 16 * c, o);
                }
            }
            if (my_ref != m_use) {
                l_part *= ex2(my_ref - m_safe);
                my_ref = m_use;
            }
            float ls = 0.f;
#pragma unroll
            for (int c = 0; c < kBlock; c += 64) {
                if (Q8 && q8) {
                    load_scores(sa + c, r);
                    ls = kind == kFull ? q8_exp<F16, false>(r, sa + c / 2, 0, 64, cw + c, cv + c, -m_safe, ls)
                                       : q8_exp<F16, true>(r, sa + c / 2, lo - c, hi - c, cw + c, cv + c, -m_safe, ls);
                } else {
                    t4_scores(sa + c, kind, has_empty, lo - c, hi - c, cw + c, r);
                    ls = kind == kFar ? t4_exp<true, F16>(r, sa + c / 2, cw + c, p.scale_log2, -m_safe, ls)
                                      : t4_exp<false, F16>(r, sa + c / 2, cw + c, p.scale_log2, -m_safe, ls);
                }
            }
            l_part += ls;
            if (SRC == kPages16 && it == n - 1) {
                // The value rows behind the sequence's end: the weights there are zero, what the page holds need not be a number.
                const int valid = tile.n - tile.pos0 / kBlock * kBlock;
                if (valid < kBlock) {
                    constexpr int per = 2;                    // the last load of the ring is this item's value tile
                    const int vslot = (per * n - 1) % NS;
                    if (!__all_sync(kAll, mbar_wait(&kv_full[vslot], ((per * n - 1) / NS) & 1, p.wait_limit))) {
                        ok = false;
                        break;
                    }
                    if (row >= valid) {
#pragma unroll
                        for (int h = 0; h < NH; ++h)
#pragma unroll
                            for (int x = 0; x < 8; ++x)
                                *reinterpret_cast<uint4 *>(smem + C::kRing + vslot * C::kTile + h * kHalfBytes + row * 128 + 16 * x) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[g]);
        }
        // ---- merge the partial denominators, O / l once the last product has finished
        s_lend[g][row] = l_part;
        s_mend[g][row] = my_ref;
        __syncwarp();
        if (lane == 0) mbar_arrive(&endbar);
        if (ok && !__all_sync(kAll, mbar_wait(&endbar, 0, p.wait_limit))) ok = false;
        if (ok && !__all_sync(kAll, mbar_wait(&pv_done[(n - 1) % NB], ((n - 1) / NB) & 1, p.wait_limit))) ok = false;
        tc_fence_after();
        if (!ok) s_err = 1;
        if (ok && g < 2) {
            const float ref = s_ref[row];
            float den = 0.f;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const float li = s_lend[i][row];
                if (li != 0.f) den += li * ex2(s_mend[i][row] - ref);
            }
            const float inv = den != 0.f ? 1.f / den : 0.f;
            uint32_t r[C::kOq];
#pragma unroll
            for (int c = 0; c < C::kOq / 32; ++c) tmem_ld32(o_addr + g * C::kOq + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&r[32 * c]));
            tc_wait_ld();
            // the warp's 32 rows through the tile ring (every read of it has finished) and out in whole lines, eight lanes a row
            constexpr int kRowB = C::kOq * 2, kPitch = kRowB + 16;
            uint8_t *stg = smem + C::kRing + warp * (32 * kPitch);
#pragma unroll
            for (int j = 0; j < C::kOq / 8; ++j) {
                uint4 w;
                w.x = pack16<F16>(__uint_as_float(r[8 * j]) * inv, __uint_as_float(r[8 * j + 1]) * inv);
                w.y = pack16<F16>(__uint_as_float(r[8 * j + 2]) * inv, __uint_as_float(r[8 * j + 3]) * inv);
                w.z = pack16<F16>(__uint_as_float(r[8 * j + 4]) * inv, __uint_as_float(r[8 * j + 5]) * inv);
                w.w = pack16<F16>(__uint_as_float(r[8 * j + 6]) * inv, __uint_as_float(r[8 * j + 7]) * inv);
                *reinterpret_cast<uint4 *>(stg + lane * kPitch + 16 * j) = w;
            }
            __syncwarp();
            constexpr int kLanesPerRow = kRowB / 16, kRowsPerIt = 32 / kLanesPerRow;
            const int sub = lane / kLanesPerRow, ch = lane % kLanesPerRow, valid = tile.ntok * p.G;
            T *obase = static_cast<T *>(p.out) + g * C::kOq + 8 * ch;
#pragma unroll
            for (int x = 0; x < 32 / kRowsPerIt; ++x) {
                const int rr = x * kRowsPerIt + sub, qr = lq * 32 + rr;
                const uint4 w = *reinterpret_cast<const uint4 *>(stg + rr * kPitch + 16 * ch);
                if (qr < valid) {
                    const int64_t t = tile.t0 + qr / p.G, h = hk * p.G + qr % p.G;
                    *reinterpret_cast<uint4 *>(obase + t * p.o_t + h * p.o_h) = w;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (s_err && tid == 0) {
        if (p.seqs.status) atomicExch(p.seqs.status, VQ_WORD_TIMEOUT);
        // a bounded wait expired: give tile loads still in flight time to land before leaving
#pragma unroll 1
        for (int w = 0; w < (1 << 14); ++w) __nanosleep(256);
    }
    __syncthreads();
    if (warp == C::kWarpLoad) {
        __syncwarp();
        tmem_dealloc(tmem, C::kCols);
    }
}

// tokens [T, Hq, D] in boxes of 64 columns x G heads x TQ tokens
static bool map_tokens(CUtensorMap *out, const void *ptr, int64_t T, const PagedAttnParams &p, int64_t s_t, int64_t s_h, int TQ, bool f16)
{
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dim[3] = {static_cast<cuuint64_t>(p.D), static_cast<cuuint64_t>(p.Hq), static_cast<cuuint64_t>(T)};
    // a dimension of one element may come with any stride: give the map one it accepts
    const cuuint64_t str[2] = {static_cast<cuuint64_t>(p.Hq > 1 ? s_h * 2 : p.D * 2), static_cast<cuuint64_t>(T > 1 ? s_t * 2 : p.Hq * p.D * 2)};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.G), static_cast<cuuint32_t>(TQ)}, es[3] = {1, 1, 1};
    return fn(out, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(ptr), dim, str, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// pool [NP, Hkv, P, D] in boxes of one page: 64 columns of 16 bits, swizzled, or whole rows of 8 bits as they are
template <bool Q8>
static bool map_pool(CUtensorMap *out, const PagedPool &pool, const PagedAttnParams &p, bool f16)
{
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return false;
    const int P = 1 << p.seqs.log_p, e = Q8 ? 1 : 2;
    const cuuint64_t dim[4] = {static_cast<cuuint64_t>(p.D), static_cast<cuuint64_t>(P), static_cast<cuuint64_t>(p.Hkv), static_cast<cuuint64_t>(p.seqs.NP)};
    const cuuint64_t str[3] = {static_cast<cuuint64_t>(pool.s_row * e), static_cast<cuuint64_t>((p.Hkv > 1 ? pool.s_head : pool.s_row) * e),
                               static_cast<cuuint64_t>((p.seqs.NP > 1 ? pool.s_page : pool.s_row) * e)};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(Q8 ? p.D : 64), static_cast<cuuint32_t>(P), 1, 1}, es[4] = {1, 1, 1, 1};
    return fn(out, Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
              const_cast<void *>(pool.ptr), dim, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, Q8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Blocks of 128 keys of a call's sequences, from the first that a new token sees on: codes -> 16-bit floats (exact; half values times the power of two
// that goes with their row's scale), rows behind the end -> zeros.  A CTA per block, kv head and pool; bound by memory traffic.
template <typename T, int D>
__global__ void __launch_bounds__(256) convert_blocks_kernel(const PagedAttnParams p)
{
    __shared__ int s_seq, s_blk, s_n, s_last;
    const int tid = threadIdx.x, lane = tid & 31, hk = blockIdx.y, pool_id = blockIdx.z;      // 0: k1, 1: v, 2: k3
    if (tid < 32) {
        int before = 0, seq = -1, blk = 0, len = 0, last = 0;
        for (int base = 0; base < p.seqs.S; base += 32) {
            int t0 = 0, q = 0, n = 0, blocks = 0, first = 0;
            if (base + lane < p.seqs.S && p.seqs.seq(base + lane, t0, q, n, p.max_q) && q > 0) {
                first = p.first_block(n - q);
                blocks = (n - 1) / kBlock - first + 1;
            }
            int sum = blocks;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(~0u, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned mine = __ballot_sync(~0u, before + sum > static_cast<int>(blockIdx.x));
            if (mine) {
                const int l = __ffs(mine) - 1;
                seq = base + l;
                blk = __shfl_sync(~0u, first, l) + static_cast<int>(blockIdx.x) - (before + __shfl_sync(~0u, sum, l) - __shfl_sync(~0u, blocks, l));
                len = __shfl_sync(~0u, n, l);
                last = (len - 1) / kBlock;
                break;
            }
            before += __shfl_sync(~0u, sum, 31);
        }
        if (lane == 0) {
            s_seq = seq;
            s_blk = blk;
            s_n = len;
            s_last = last;
        }
    }
    __syncthreads();
    const int seq = s_seq, blk = s_blk, n = s_n;
    if (seq < 0 || (pool_id == 2 && blk > s_last - p.W / kBlock)) return;      // raw keys: those before somebody's exact window
    const PagedPool &pool = pool_id == 0 ? p.k1 : pool_id == 1 ? p.v : p.k3;
    const int page_mask = (1 << p.seqs.log_p) - 1;
    constexpr bool kHalf = !IsBf16<T>::value;
    const int64_t at = (pool_id * p.ws_blocks + blockIdx.x) * p.Hkv + hk;
    if (tid < kBlock) {                                      // what multiplies the scores of a key, or the weights of a value
        const int key = blk * kBlock + tid, page = key < n ? p.seqs.page(seq, key >> p.seqs.log_p) : -1;
        const float x = page >= 0 ? __ldg(pool.scale + pool.scale_at(page, hk, key & page_mask)) : 0.f;
        float p2;
        p.ws_scales(3 * p.ws_blocks * p.Hkv * (kBlock * D * 2))[at * kBlock + tid] =
            pool_id != 1 ? x * p.scale_log2 : kHalf ? half_weight_factor(x, p2) : x;
    }
    T *dst = static_cast<T *>(p.ws) + at * (kBlock * D);
    constexpr int CH = D / 16;
#pragma unroll
    for (int x = tid; x < kBlock * CH; x += 256) {
        const int row = x / CH, c = x % CH * 16, key = blk * kBlock + row;
        uint4 codes = make_uint4(0, 0, 0, 0), a, b;
        const int page = key < n ? p.seqs.page(seq, key >> p.seqs.log_p) : -1;
        if (page >= 0) codes = *reinterpret_cast<const uint4 *>(static_cast<const int8_t *>(pool.ptr) + pool.row(page, hk, key & page_mask) + c);
        if constexpr (IsBf16<T>::value) {
            Codes8<T>::expand(codes.x, a.x, a.y);
            Codes8<T>::expand(codes.y, a.z, a.w);
            Codes8<T>::expand(codes.z, b.x, b.y);
            Codes8<T>::expand(codes.w, b.z, b.w);
        } else {
            const float scale = pool_id == 1 && page >= 0 ? __ldg(pool.scale + pool.scale_at(page, hk, key & page_mask)) : 0.f;
            const __half2 m2 = __float2half2_rn(pool_id == 1 ? pow2f(-half_weight_shift(scale)) : 1.f);
            Codes8<T>::expand_scaled(codes.x, m2, a.x, a.y);
            Codes8<T>::expand_scaled(codes.y, m2, a.z, a.w);
            Codes8<T>::expand_scaled(codes.z, m2, b.x, b.y);
            Codes8<T>::expand_scaled(codes.w, m2, b.z, b.w);
        }
        *reinterpret_cast<uint4 *>(dst + row * D + c) = a;
        *reinterpret_cast<uint4 *>(dst + row * D + c + 8) = b;
    }
}

template <int D, bool F16, int SRC>
static int launch_chunk(const PagedAttnParams &a, cudaStream_t stream)
{
    using C = ChunkCfg<D, SRC == kPages8>;
    using T = typename std::conditional<F16, __half, __nv_bfloat16>::type;
    ChunkParams cp;
    cp.a = a;
    if (SRC != kWorkspace) cp.a.ws = nullptr;
    cp.TQ = kBlock / a.G;
    TcMaps m;
    if (!map_tokens(&m.q1, a.q1, a.seqs.T, a, a.q1_t, a.q1_h, cp.TQ, F16) || !map_tokens(&m.q2, a.q2, a.seqs.T, a, a.q2_t, a.q2_h, cp.TQ, F16)) return VQ_ELAUNCH;
    if (SRC == kWorkspace) {
        const uint64_t wd[3] = {D, kBlock, static_cast<uint64_t>(a.ws_blocks) * a.Hkv}, wst[3] = {1, D, kBlock * D};
        const int64_t per = a.ws_blocks * a.Hkv * (kBlock * D);
        T *ws = static_cast<T *>(a.ws);
        if (!make_map(&m.k1, ws, 3, wd, wst, kBlock, F16) || !make_map(&m.v, ws + per, 3, wd, wst, kBlock, F16) ||
            !make_map(&m.k3, a.rerope ? ws + 2 * per : ws, 3, wd, wst, kBlock, F16))
            return VQ_ELAUNCH;
        const dim3 grid(static_cast<unsigned>(a.ws_blocks), static_cast<unsigned>(a.Hkv), a.rerope ? 3u : 2u);
        convert_blocks_kernel<T, D><<<grid, 256, 0, stream>>>(cp.a);
        const int st = launch_status();
        if (st != VQ_OK) return st;
    } else if (!map_pool<SRC != kPages16>(&m.k1, a.k1, a, F16) || !map_pool<SRC != kPages16>(&m.k3, a.k3, a, F16) ||
               !map_pool<SRC != kPages16>(&m.v, a.v, a, F16)) {
        return VQ_ELAUNCH;
    }
    if (a.cb != nullptr) {
        const uint64_t MK = a.MK, cd[3] = {D, MK, static_cast<uint64_t>(a.Hkv)}, cs[3] = {1, D, MK * D}, vd[3] = {D, MK, static_cast<uint64_t>(a.NS) * a.Hkv};
        if (!make_map(&m.cb, a.cb, 3, cd, cs, kBlock, F16) || !make_map(&m.vs, a.vsum, 3, vd, cs, kBlock, F16)) return VQ_ELAUNCH;
    } else {
        m.cb = m.vs = m.q1;         // never read: no tile has codes
    }
    auto kern = paged_chunk_kernel<D, F16, SRC>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal) != cudaSuccess) return VQ_ELAUNCH;
    const int64_t tiles = chunk_tiles(a.seqs, cp.TQ);
    kern<<<dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(a.Hkv)), C::kThreads, C::kTotal, stream>>>(m.q1, m.q2, m.k1, m.k3, m.v, m.cb, m.vs, cp);
    return launch_status();
}

template <int D, bool F16>
static int launch_chunk_src(const PagedAttnParams &p, bool q8, cudaStream_t stream)
{
    if (!q8) return launch_chunk<D, F16, kPages16>(p, stream);
    return p.ws != nullptr ? launch_chunk<D, F16, kWorkspace>(p, stream) : launch_chunk<D, F16, kPages8>(p, stream);
}

template <bool F16>
static int launch_chunk_type(const PagedAttnParams &p, bool q8, cudaStream_t stream)
{
    return p.D == 64 ? launch_chunk_src<64, F16>(p, q8, stream) : launch_chunk_src<128, F16>(p, q8, stream);
}

int launch_paged_chunk(const PagedAttnParams &p, int dtype, bool q8, cudaStream_t stream)
{
    return dtype == VQ_F16 ? launch_chunk_type<true>(p, q8, stream) : launch_chunk_type<false>(p, q8, stream);
}

}  // namespace vq
