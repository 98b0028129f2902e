// Attention over a paged cache for few new tokens per sequence (one token of a decode, a handful of drafted ones): at most 32 query rows -
// tokens times query heads - share a kv head's keys.
//
// Bound by HBM: 4 D operations per key and row against 4 D (2 D) bytes per key.  So the work is organised around the stream of rows, and the
// matrix product only has to keep out of its way: mma.sync with the KEYS on the M axis (16 per instruction) and 8 query rows on N, for
// which a tile of 128 rows of tcgen05 would be nearly empty.  A warp takes steps of 16 keys (32 of 8-bit rows) and keeps its own online
// softmax: no barrier in the loop.
//   - A warp's keys and values arrive by TMA, 16 rows a box, in a FIFO of its own, filled by one more warp of the CTA (no CTA barrier).  Both products may
//     permute their reduction index: a thread reads 16 contiguous bytes of a swizzled key row, which hold its operands of several k-steps, and q
//     is read in the same order.  Values enter as V^T (D on M): pairs of keys are interleaved by byte permutes.
//   - S^T (keys x rows) becomes the B operand of the second product by movmatrix, 8 x 8 at a time.
//   - 8-bit codes become halves exactly (byte permutes and a subtraction).  A key's scale multiplies its score.  A bf16 query row is brought into
//     the range of a half by a power of two (its largest element to 2^10 .. 2^11; elements above 2^-24 of it stay exact).  Weights carry the
//     scale of their value.
//   - Counts multiply the weights of codes in the denominator; codes without members are excluded.
//   - Weights are rounded to 16 bits before they meet their values, as the matrix instruction wants both in one type (and as the prefill kernels do);
//     their sum is not.  It costs as much as rounding the output: 2.3e-3 of the result (bf16, against 64 bits) where that alone is 1.7e-3.
// One unit = (sequence, block of positions, kv head); its steps are dealt out to the warps of a cluster of 1 - 16 CTAs, which merge their
// partial sums through distributed shared memory: no workspace, no second launch, the same order of additions every time.
#include <cooperative_groups.h>
#include <type_traits>

#include "codes8.cuh"
#include "paged_attn.cuh"
#include "prefill_tc_common.cuh"
#include "tc_ptx.cuh"

namespace vq {

namespace cg = cooperative_groups;

constexpr int kFewSplit = 16;           // CTAs of a cluster at most (more than 8 are opt-in on this architecture)
constexpr float kFewLazy = 8.f;         // log2 units a score may exceed its row's reference before the sums are rescaled

template <typename T> struct Mma16816;
template <> struct Mma16816<__nv_bfloat16> {
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct Mma16816<__half> {
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
__device__ __forceinline__ uint32_t movmatrix(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T, bool Q8, int D, int NT>
struct FewCfg {
    // Warps that compute (one more issues the loads), stages of their FIFOs, CTAs of an SM: what registers and shared memory allow.  Measured, us.
    // Up to 8 rows: 64 sequences of 8 kv heads, 16 bits, 3 warps x 2 stages x 4 CTAs / 4 x 3 x 2: 136 / 152 (all 512 units run at once); 16
    // sequences of 32 heads, 8 bits, 5 x 2 x 2 / 4 x 3 x 2 / 3 x 2 x 3: 77 / 87 / 104.  16 rows, 32 sequences of 8 heads, D = 128, 3 x 3 x 2 /
    // 4 x 3 x 2 (8 bits: 5 x 3 x 2): 46 / 50, 8 bits 64 / 90 (which spills); D = 64: 42 / 38, 45 / 34.  32 rows, 7 x 2 x 1 / 4 x 3 x 1: 94 / 123,
    // 8 bits 125 / 144, D = 64 68 / 74.  With D = 128 that form spills 0.4 KB a thread (8 bits: 1 KB): four column tiles of sums, their operands
    // and a step's rows are more than 255 registers.
    static constexpr int kWarps = NT == 1 ? (Q8 ? 5 : 3) : NT == 2 ? (D == 128 ? 3 : Q8 ? 5 : 4) : 7, kThreads = (kWarps + 1) * 32;
    static constexpr int kStages = NT == 2 ? 3 : 2;
    static constexpr int kCtas = NT == 1 ? (Q8 ? 2 : 4) : NT == 2 ? 2 : 1;
    static constexpr int kCols = 8 * NT;                         // query rows, padded
    static constexpr int VC = D / 64;                            // boxes of 64 columns of a 16-bit row
    static constexpr int kBox = 16 * 128;                        // bytes of 16 rows x 64 columns of 16 bits
    static constexpr int kBox8 = 16 * D;                         // 16 rows of 8 bits
    static constexpr int kStage = 2 * VC * kBox;                 // 16 keys with their values, or 32 of 8 bits
    static_assert(4 * kBox8 == kStage, "a stage holds twice as many 8-bit rows");
    static constexpr int kWarpBytes = kStages * kStage;
    static constexpr int kQ = (Q8 ? 3 : 2) * kCols * D * 2;      // rows q1, q2; 8-bit rows: q2, and both as halves
    static constexpr int kPages = 256;                           // page table entries kept in shared memory; the rest is read where it is needed
    static constexpr int kTotal = kWarps * kWarpBytes + kQ + kPages * 4 + 1024;   // + slack for 1024-byte alignment
    static_assert(kCols * D * 4 <= kStages * kStage, "a warp's sums fit into its FIFO");
    // Log2 units that a row's reference lies below the score that set it.  Weights meet their values in 16 bits: a half loses bits below 2^-14, which
    // half caches have anyway, but a bf16 does not.  So the halves of a bf16 cache with 8-bit rows use the upper end of their range: up to
    // 2^(8 + 6) times a factor below 2, all bits down to 2^-20 of the largest weight.
    static constexpr float kBelow = Q8 && IsBf16<T>::value ? 6.f : 0.f;
    static constexpr int MT = D / 16;
};

struct FewSteps {
    int n_far, n_old, n_near;       // steps of codes, of raw keys before the exact window, of rotated keys
    int old0, near0;                // first key of the latter two (multiples of 16)
};

template <typename T, bool Q8, int D, int NT>
__global__ void __launch_bounds__(FewCfg<T, Q8, D, NT>::kThreads, FewCfg<T, Q8, D, NT>::kCtas)
paged_few_kernel(const __grid_constant__ CUtensorMap tm_k1, const __grid_constant__ CUtensorMap tm_k3, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ CUtensorMap tm_cb, const __grid_constant__ CUtensorMap tm_vs, const PagedAttnParams p, int nsplit)
{
    using C = FewCfg<T, Q8, D, NT>;
    using M = Mma16816<T>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-ptx::smem_u32(smem_raw) & 1023u);   // stays an address of shared memory for the compiler
    __shared__ __align__(8) uint64_t s_bar[C::kWarps][C::kStages], s_free[C::kWarps][C::kStages];
    __shared__ int s_bad;                                            // some page of the unit is missing, or not kept in shared memory
    __shared__ float s_m[C::kWarps][C::kCols], s_l[C::kWarps][C::kCols];
    __shared__ float s_cm[C::kCols], s_cl[C::kCols];
    __shared__ float s_unit[2][Q8 ? C::kCols : 1];                   // 8-bit rows: the power of two a query row was divided by
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = lane >> 2, c = lane & 3;
    T *s_q = reinterpret_cast<T *>(smem + C::kWarps * C::kWarpBytes);        // [2][kCols][D]
    __half *s_qh = reinterpret_cast<__half *>(s_q + C::kCols * D);           // 8-bit rows: [q1, q2][kCols][D]
    int *s_page = reinterpret_cast<int *>(smem + C::kWarps * C::kWarpBytes + C::kQ);

    const int split = blockIdx.x % nsplit;
    int unit = blockIdx.x / nsplit;
    const int hk = unit % p.Hkv;
    unit /= p.Hkv;
    const int s = unit % p.seqs.S, grp = unit / p.seqs.S;           // second blocks, hardly ever there, come last: the others get an SM each
    int t0, q, n;
    grid_dependency_launch();
    grid_dependency_wait();
    if (!p.seqs.seq(s, t0, q, n, p.max_q) || q == 0) return;         // the whole cluster leaves
    int i0 = n - q, i1 = n - 1;                                      // positions of the group's tokens: those of one 128-block
    if (grp == 0) i1 = min(i1, i0 / kBlock * kBlock + kBlock - 1);
    else {
        const int next = i0 / kBlock * kBlock + kBlock;
        t0 += next - i0;
        i0 = next;
        if (i0 > i1) return;
    }
    const int rows = (i1 - i0 + 1) * p.G;
    const int bd = p.boundary(i0), entry = p.snapshot_entry(s, bd);
    FewSteps st;
    constexpr bool kHalf = Q8 && !IsBf16<T>::value;
    constexpr int KEYS = Q8 ? 32 : 16;                               // keys per step of window rows
    st.old0 = bd;
    const int old_end = p.rerope ? max(0, i1 - p.W) : 0;             // raw keys: [bd, old_end)
    st.n_old = old_end > bd ? (old_end - bd + KEYS - 1) / KEYS : 0;
    st.near0 = (p.rerope ? max(0, i0 - p.W) : bd) & ~15;
    st.n_near = (i1 - st.near0) / KEYS + 1;
    int snap = -1, total = 0;
    auto plan = [&]() {                                              // uses the table's entry, which has been under way since
        snap = p.checked_snapshot(bd, entry);
        st.n_far = snap >= 0 ? p.MK / 16 : 0;
        total = st.n_far + st.n_old + st.n_near;
    };
    const int col0 = bd >> p.seqs.log_p, cols = (i1 >> p.seqs.log_p) - col0 + 1;

    // The other warps fetch the query rows while the loading warp (below) sets up the barriers and the page table and goes ahead; they meet at a
    // named barrier where that one does not stop.
    if (warp != C::kWarps) {
        // ---- query rows.  Rows behind `rows` are zeros.
        auto q_row = [&](int which, int row) {
            const int64_t t = t0 + row / p.G, h = hk * p.G + row % p.G;
            return which ? static_cast<const T *>(p.q2) + t * p.q2_t + h * p.q2_h : static_cast<const T *>(p.q1) + t * p.q1_t + h * p.q1_h;
        };
        for (int x = tid; x < (Q8 ? 1 : 2) * C::kCols * D / 8; x += C::kWarps * 32) {
            const int which = Q8 ? 1 : x / (C::kCols * D / 8), row = x / (D / 8) % C::kCols, d = x % (D / 8) * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < rows) v = *reinterpret_cast<const uint4 *>(q_row(which, row) + d);
            reinterpret_cast<uint4 *>(s_q)[x] = v;
        }
        if constexpr (Q8) {
            for (int x = warp; x < 2 * C::kCols; x += C::kWarps) {
                const int which = x / C::kCols, row = x % C::kCols;
                float e[D / 32], top = 0.f;
                int shift = 0;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) e[i] = 0.f;
                if (row < rows) {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        e[i] = to_f32(q_row(which, row)[lane * (D / 32) + i]);
                        top = fmaxf(top, fabsf(e[i]));
                    }
                    if constexpr (IsBf16<T>::value) {
#pragma unroll
                        for (int y = 16; y; y >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, y));
                        const int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
                        if (top > 0.f && ex < 128) shift = max(-100, ex) - 10;
                    }
                }
                const float mul = __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll
                for (int i = 0; i < D / 32; i += 2)
                    *reinterpret_cast<__half2 *>(s_qh + (which * C::kCols + row) * D + lane * (D / 32) + i) = __floats2half2_rn(e[i] * mul, e[i + 1] * mul);
                if (lane == 0) s_unit[which][row] = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
            }
        }
    }
    plan();

    const int64_t far_base = (static_cast<int64_t>(snap < 0 ? 0 : snap) * p.Hkv + hk) * p.MK;
    const int page_mask = (1 << p.seqs.log_p) - 1;
    auto page_of = [&](int j) {
        const int x = (j >> p.seqs.log_p) - col0;
        return x < C::kPages ? s_page[x] : p.seqs.page(s, x + col0);
    };
    auto first_key = [&](int step) {
        return step < st.n_far + st.n_old ? st.old0 + (step - st.n_far) * KEYS : st.near0 + (step - st.n_far - st.n_old) * KEYS;
    };
    // ---- keys and values of a step into stage `slot` of warp w, by one thread.  Missing pages (reported) bring nothing.
    auto fill = [&](int w, int step, int slot) {
        uint8_t *dst = smem + w * C::kWarpBytes + slot * C::kStage;
        uint64_t *bar = &s_bar[w][slot];
        if (step < st.n_far) {
            ptx::mbar_expect_tx(bar, C::kStage);
#pragma unroll
            for (int h = 0; h < C::VC; ++h) {
                ptx::tma_load_3d(dst + h * C::kBox, &tm_cb, bar, 64 * h, step * 16, hk);
                ptx::tma_load_3d(dst + (C::VC + h) * C::kBox, &tm_vs, bar, 64 * h, step * 16, snap * p.Hkv + hk);
            }
            return;
        }
        const CUtensorMap *tm = step < st.n_far + st.n_old ? &tm_k3 : &tm_k1;
        const int key0 = first_key(step);
        int pg[KEYS / 16], some = 0;
#pragma unroll
        for (int u = 0; u < KEYS / 16; ++u) {
            pg[u] = key0 + 16 * u <= i1 ? page_of(key0 + 16 * u) : -1;
            some += pg[u] >= 0;
        }
        ptx::mbar_expect_tx(bar, some * (C::kStage / (KEYS / 16)));
#pragma unroll
        for (int u = 0; u < KEYS / 16; ++u) {
            const int pr = (key0 + 16 * u) & page_mask;
            if (pg[u] < 0) continue;
            if constexpr (Q8) {
                ptx::tma_load_4d(dst + 2 * u * C::kBox8, tm, bar, 0, pr, hk, pg[u]);
                ptx::tma_load_4d(dst + (2 * u + 1) * C::kBox8, &tm_v, bar, 0, pr, hk, pg[u]);
            } else {
#pragma unroll
                for (int h = 0; h < C::VC; ++h) {
                    ptx::tma_load_4d(dst + h * C::kBox, tm, bar, 64 * h, pr, hk, pg[u]);
                    ptx::tma_load_4d(dst + (C::VC + h) * C::kBox, &tm_v, bar, 64 * h, pr, hk, pg[u]);
                }
            }
        }
    };
    // ---- what goes with the rows: lane l has the count of code l, or the scales of key l and of its value
    auto extras = [&](int step, float &x, float &y) {
        x = y = 0.f;
        if (step >= total) return;
        if (step < st.n_far) {
            x = __ldg(p.cnt + far_base + step * 16 + (lane & 15));
        } else if constexpr (Q8) {
            const int j = first_key(step) + lane;
            const bool in = j < n && j <= (i1 | 15), old = step < st.n_far + st.n_old;
            const int pg = in ? page_of(j) : -1, page = max(pg, 0), pr = j & page_mask;
            const float *ks = old ? p.k3.scale + p.k3.scale_at(page, hk, pr) : p.k1.scale + p.k1.scale_at(page, hk, pr);
            x = __ldg(ks);
            y = __ldg(p.v.scale + p.v.scale_at(page, hk, pr));
            if (!(fabsf(y) < INFINITY)) {                            // a value row that is not finite: its score says so to the tokens that see it,
                x = __int_as_float(0x7fffffff);                      // and the others do not multiply it by zero
                y = 0.f;
            }
            if (pg < 0) x = y = 0.f;
        }
    };

    const int stride = nsplit * C::kWarps;
    bool failed = false;
    if (warp == C::kWarps) {
        if (lane == 0) {
            for (int w = 0; w < C::kWarps; ++w)
                for (int x = 0; x < C::kStages; ++x) {
                    ptx::mbar_init(&s_bar[w][x], 1);
                    ptx::mbar_init(&s_free[w][x], 1);
                }
            ptx::fence_mbar_init();
        }
        __syncwarp();
        // Lane w looks after warp w's FIFO: step and stage of its next fill.  Those that find their stage free are served one after another by
        // one elected thread; nobody waits for a warp that is behind.
        int step = lane < C::kWarps ? split * C::kWarps + lane : total, fills = 0, slot = 0;
        uint32_t par = 1u;
        auto serve = [&](bool ready) {
            for (unsigned left = __ballot_sync(~0u, ready); left; left &= left - 1) {
                const int w = __ffs(left) - 1, at = __shfl_sync(~0u, step, w), to = __shfl_sync(~0u, slot, w);
                if (ptx::elect_one()) fill(w, at, to);
                __syncwarp();
            }
            if (!ready) return;
            step += stride;
            ++fills;
            if (++slot == C::kStages) {
                slot = 0;
                par ^= 1u;
            }
        };
#pragma unroll 1
        for (int x = 0; x < C::kStages; ++x) serve(step < st.n_far);  // codes need no page table
        bool miss = cols > C::kPages;
        for (int x = lane; x < min(cols, C::kPages); x += 32) {
            const int pg = p.seqs.page(s, col0 + x);
            s_page[x] = pg;
            miss = miss || pg < 0;
        }
        miss = __any_sync(~0u, miss);
        if (lane == 0) s_bad = miss;
        __syncwarp();
        asm volatile("bar.arrive 1, %0;" ::"n"(C::kThreads) : "memory");
        long long since = clock64();
        while (__any_sync(~0u, step < total)) {
            const bool ready = step < total && (fills < C::kStages || ptx::mbar_test(&s_free[lane][slot], par));
            if (__any_sync(~0u, ready)) {
                serve(ready);
                since = clock64();
            } else if (clock64() - since > p.wait_limit) {
                failed = true;
                break;
            }
        }
    } else {
        float o[NT][C::MT][4], m[NT][2], lim[NT][2], l[NT][2], qu[NT][2];   // lim: the score that raises the reference m
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[nt][mt][x] = 0.f;
            m[nt][0] = m[nt][1] = lim[nt][0] = lim[nt][1] = -INFINITY;
            qu[nt][0] = qu[nt][1] = 0.f;
            l[nt][0] = l[nt][1] = 0.f;
        }
        uint32_t qf[NT][D / 8];
        uint8_t *const fifo = smem + warp * C::kWarpBytes;
        const int first = split * C::kWarps + warp;
        asm volatile("bar.sync 1, %0;" ::"n"(C::kThreads) : "memory");
        const bool bad = s_bad;
        float next_x, next_y;
        extras(first, next_x, next_y);
        // sc: scores of keys r and r + 8 of each group of 16 (c0 c1 | c2 c3) in log2 units, -inf where excluded -> weights; w: denominator weights of
        // the two keys, f: factors of their value rows.  Raises the references, adds to l, returns the packed weights as B operands.
        auto softmax = [&](auto &sc, const auto &w, const auto &f, auto &pb, bool half) {
            constexpr int SUBS = sizeof(sc) / sizeof(sc[0]);
            bool above = false;
            float mx[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mx[nt][x] = fmaxf(sc[0][nt][x], sc[0][nt][2 + x]);
#pragma unroll
                    for (int u = 1; u < SUBS; ++u) mx[nt][x] = ptx::fmax3(mx[nt][x], sc[u][nt][x], sc[u][nt][2 + x]);
                    above |= mx[nt][x] > lim[nt][x];
                }
            if (__any_sync(~0u, above)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float v = mx[nt][x];
#pragma unroll
                        for (int y = 4; y < 32; y <<= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, y));
                        const float ref = v - C::kBelow;
                        if (ref > m[nt][x]) {
                            const float a = m[nt][x] == -INFINITY ? 0.f : ptx::ex2(m[nt][x] - ref);
                            m[nt][x] = ref;
                            lim[nt][x] = v + kFewLazy;
                            l[nt][x] *= a;
#pragma unroll
                            for (int mt = 0; mt < C::MT; ++mt) {
                                o[nt][mt][x] *= a;
                                o[nt][mt][2 + x] *= a;
                            }
                        }
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float ma = m[nt][0] == -INFINITY ? 0.f : m[nt][0], mb = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
                for (int u = 0; u < SUBS; ++u) {
                    const float p0 = ptx::ex2(sc[u][nt][0] - ma), p1 = ptx::ex2(sc[u][nt][1] - mb), p2 = ptx::ex2(sc[u][nt][2] - ma), p3 = ptx::ex2(sc[u][nt][3] - mb);
                    l[nt][0] += p0 * w[u][0] + p2 * w[u][1];
                    l[nt][1] += p1 * w[u][0] + p3 * w[u][1];
                    const float a0 = p0 * f[u][0], a1 = p1 * f[u][0], a2 = p2 * f[u][1], a3 = p3 * f[u][1];
                    pb[u][nt][0] = movmatrix(half ? ptx::pack_f16(a0, a1) : Pair16<T>::pack(a0, a1));
                    pb[u][nt][1] = movmatrix(half ? ptx::pack_f16(a2, a3) : Pair16<T>::pack(a2, a3));
                }
            }
        };
        // excluded keys of the 16 from j0 on; true: there is no such page (bad: some page is missing)
        auto mask = [&](float (&sc)[NT][4], int j0, bool old) {
            if (bad && j0 <= i1 && page_of(j0) < 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[nt][x] = -INFINITY;
                return true;
            }
            // what every row of the group sees: raw keys below i0 - W, rotated ones in [i1 - W, i0]
            const bool all = old ? j0 + 15 < i0 - p.W : j0 + 15 <= i0 && (!p.rerope || j0 >= i1 - p.W);
            if (all) return false;
            const int ja = j0 + r, jb = ja + 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int i = i0 + (8 * nt + 2 * c + x) / p.G, hi = old ? i - p.W - 1 : i, lo = old || !p.rerope ? bd : i - p.W;
                    if (ja < lo || ja > hi || ja >= n) sc[nt][x] = -INFINITY;
                    if (jb < lo || jb > hi || jb >= n) sc[nt][2 + x] = -INFINITY;
                }
            return false;
        };

        int phase = -1, slot = 0;
        uint32_t par = 0;
        for (int step = first; step < total; step += stride) {
            const bool far = step < st.n_far, old = !far && step < st.n_far + st.n_old;
            const int ph = far ? 0 : old ? 1 : 2;
            if (ph != phase) {                                           // q in the order of this phase's key rows
                phase = ph;
                if (Q8 && !far) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const __half *row = s_qh + ((old ? C::kCols : 0) + 8 * nt + r) * D + 16 * C::VC * c;
#pragma unroll
                        for (int j = 0; j < 2 * C::VC; ++j) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(row + 8 * j);
                            qf[nt][4 * j] = v.x; qf[nt][4 * j + 1] = v.y; qf[nt][4 * j + 2] = v.z; qf[nt][4 * j + 3] = v.w;
                        }
#pragma unroll
                        for (int x = 0; x < 2; ++x) qu[nt][x] = s_unit[old][8 * nt + 2 * c + x] * p.scale_log2;
                    }
                } else {
                    const T *src = s_q + (!Q8 && (far || old) ? C::kCols * D : 0);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2 * C::VC; ++j) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(src + (8 * nt + r) * D + 64 * (j / 2) + 16 * c + 8 * (j % 2));
                            qf[nt][4 * j] = v.x; qf[nt][4 * j + 1] = v.y; qf[nt][4 * j + 2] = v.z; qf[nt][4 * j + 3] = v.w;
                        }
                }
            }
            const float my_x = next_x, my_y = next_y;
            extras(step + stride, next_x, next_y);
            const uint8_t *stg = fifo + slot * C::kStage;
            if (!__all_sync(~0u, ptx::mbar_wait(&s_bar[warp][slot], par, p.wait_limit))) {
                failed = true;
                break;
            }
            const int key0 = first_key(step);
            if (far || !Q8) {
                // ---- S^T = K Q^T, even and odd k-steps by themselves.  Piece j of row k lies at j ^ (k % 8); four lanes share a row, each
                // takes two neighbouring pieces of its 128 bytes: the eight lanes that read together ask for different banks.
                // All reads come first: what follows is code without branches but for the rare ones.
                uint4 ka[2 * C::VC], kb[2 * C::VC], v4[C::VC][4];
#pragma unroll
                for (int j = 0; j < 2 * C::VC; ++j) {
                    const uint8_t *at = stg + (j / 2) * C::kBox + r * 128 + (((2 * c + j % 2) ^ r) << 4);
                    ka[j] = *reinterpret_cast<const uint4 *>(at);
                    kb[j] = *reinterpret_cast<const uint4 *>(at + 8 * 128);
                }
#pragma unroll
                for (int h = 0; h < C::VC; ++h)
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const int k = 2 * c + (a & 1) + 8 * (a >> 1);
                        v4[h][a] = *reinterpret_cast<const uint4 *>(stg + (C::VC + h) * C::kBox + k * 128 + ((r ^ (k & 7)) << 4));
                    }
                float sc[1][NT][4], s2[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[0][nt][x] = s2[nt][x] = 0.f;
#pragma unroll
                for (int j = 0; j < 2 * C::VC; ++j)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        M::mma(sc[0][nt], ka[j].x, kb[j].x, ka[j].y, kb[j].y, qf[nt][4 * j], qf[nt][4 * j + 1]);
                        M::mma(s2[nt], ka[j].z, kb[j].z, ka[j].w, kb[j].w, qf[nt][4 * j + 2], qf[nt][4 * j + 3]);
                    }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[0][nt][x] = (sc[0][nt][x] + s2[nt][x]) * p.scale_log2;
                // codes: counts as denominator weights, those without members excluded
                const float cnt0 = __shfl_sync(~0u, my_x, r), cnt1 = __shfl_sync(~0u, my_x, r + 8);
                const float w[1][2] = {{far ? cnt0 : 1.f, far ? cnt1 : 1.f}}, f[1][2] = {{1.f, 1.f}};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (!(w[0][0] > 0.f)) sc[0][nt][0] = sc[0][nt][1] = -INFINITY;
                    if (!(w[0][1] > 0.f)) sc[0][nt][2] = sc[0][nt][3] = -INFINITY;
                }
                if (!far) {
                    const bool hole = mask(sc[0], key0, old);
                    if (hole || key0 + 16 > n) {                     // behind the sequence's end a page may hold anything: zeros instead
#pragma unroll
                        for (int h = 0; h < C::VC; ++h)
#pragma unroll
                            for (int a = 0; a < 4; ++a)
                                if (hole || key0 + 2 * c + (a & 1) + 8 * (a >> 1) >= n) v4[h][a] = make_uint4(0, 0, 0, 0);
                    }
                }
                uint32_t pb[1][NT][2];
                softmax(sc, w, f, pb, false);
                // ---- O^T += V^T P^T
#pragma unroll
                for (int h = 0; h < C::VC; ++h) {
                    const uint32_t v0[4] = {v4[h][0].x, v4[h][0].y, v4[h][0].z, v4[h][0].w}, v1[4] = {v4[h][1].x, v4[h][1].y, v4[h][1].z, v4[h][1].w};
                    const uint32_t v2[4] = {v4[h][2].x, v4[h][2].y, v4[h][2].z, v4[h][2].w}, v3[4] = {v4[h][3].x, v4[h][3].y, v4[h][3].z, v4[h][3].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t a0 = __byte_perm(v0[x], v1[x], 0x5410), a1 = __byte_perm(v0[x], v1[x], 0x7632);
                        const uint32_t a2 = __byte_perm(v2[x], v3[x], 0x5410), a3 = __byte_perm(v2[x], v3[x], 0x7632);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) M::mma(o[nt][4 * h + x], a0, a1, a2, a3, pb[0][nt][0], pb[0][nt][1]);
                    }
                }
            } else {
                // 8-bit rows of 128 (64) bytes: piece j of row k lies at j ^ (k % 8)  (j ^ (k / 2 % 4))
                auto piece = [&](int k, int j) { return D == 128 ? k * 128 + ((j ^ (k & 7)) << 4) : k * 64 + ((j ^ ((k >> 1) & 3)) << 4); };
                // Weights and values as halves: codes become halves in five instructions per four, bf16 in eight.  bf16 caches whose scales
                // leave the range of a half take the latter.
                const bool hv = kHalf || __all_sync(~0u, (my_y >= 5.9604645e-8f && my_y < 32.f) || my_y == 0.f);
                float my_p2 = 1.f;
                const float my_f = hv ? half_weight_factor(my_y, my_p2) : my_y;
                const __half2 my_pair = __floats2half2_rn(my_p2, __shfl_down_sync(~0u, my_p2, 1));   // even lanes: of keys l, l + 1
                uint4 ka[2][C::VC], kb[2][C::VC];
                uint32_t v[2][4][D / 32];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint8_t *kat = stg + 2 * u * C::kBox8, *vat = kat + C::kBox8 + 8 * (r & 1);
#pragma unroll
                    for (int j = 0; j < C::VC; ++j) {
                        ka[u][j] = *reinterpret_cast<const uint4 *>(kat + piece(r, C::VC * c + j));
                        kb[u][j] = *reinterpret_cast<const uint4 *>(kat + piece(r + 8, C::VC * c + j));
                    }
#pragma unroll
                    for (int a = 0; a < 4; ++a)
#pragma unroll
                        for (int h = 0; h < C::VC; ++h) {
                            const uint2 x = *reinterpret_cast<const uint2 *>(vat + piece(2 * c + (a & 1) + 8 * (a >> 1), 4 * h + (r >> 1)));
                            v[u][a][2 * h] = x.x; v[u][a][2 * h + 1] = x.y;
                        }
                }
                float sc[2][NT][4], s2[2][NT][4], f[2][2], w[2][2];
                __half2 p2[2][2];                                   // the powers of two that go with this thread's pairs of keys
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 4; ++x) sc[u][nt][x] = s2[u][nt][x] = 0.f;
#pragma unroll
                    for (int j = 0; j < C::VC; ++j) {
                        const uint32_t a[4] = {ka[u][j].x, ka[u][j].y, ka[u][j].z, ka[u][j].w}, b[4] = {kb[u][j].x, kb[u][j].y, kb[u][j].z, kb[u][j].w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            uint32_t al, ah, bl, bh;
                            Codes8<__half>::expand(a[x], al, ah);
                            Codes8<__half>::expand(b[x], bl, bh);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                Mma16816<__half>::mma(x & 1 ? s2[u][nt] : sc[u][nt], al, bl, ah, bh, qf[nt][8 * j + 2 * x], qf[nt][8 * j + 2 * x + 1]);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float k = __shfl_sync(~0u, my_x, 16 * u + 8 * x + r);
                        w[u][x] = 1.f;
                        f[u][x] = __shfl_sync(~0u, my_f, 16 * u + 8 * x + r);
                        p2[u][x] = __shfl_sync(~0u, my_pair, 16 * u + 8 * x + 2 * c);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            sc[u][nt][2 * x] = (sc[u][nt][2 * x] + s2[u][nt][2 * x]) * (qu[nt][0] * k);
                            sc[u][nt][2 * x + 1] = (sc[u][nt][2 * x + 1] + s2[u][nt][2 * x + 1]) * (qu[nt][1] * k);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) mask(sc[u], key0 + 16 * u, old);
                uint32_t pb[2][NT][2];
                softmax(sc, w, f, pb, hv);
                // bytes 0, 1 (y = 0) and 2, 3 of word x: m-tiles 2 x, 2 x + 1
                auto pairs = [&](int u, int x, int y, int a) { return __byte_perm(v[u][a][x], v[u][a + 1][x], y ? 0x7362 : 0x5140); };
                if (hv) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int x = 0; x < D / 32; ++x)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                uint32_t a0, a1, a2, a3;
                                Codes8<__half>::expand_scaled(pairs(u, x, y, 0), p2[u][0], a0, a1);
                                Codes8<__half>::expand_scaled(pairs(u, x, y, 2), p2[u][1], a2, a3);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) Mma16816<__half>::mma(o[nt][2 * x + y], a0, a1, a2, a3, pb[u][nt][0], pb[u][nt][1]);
                            }
                } else if constexpr (!kHalf) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int x = 0; x < D / 32; ++x)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                uint32_t a0, a1, a2, a3;
                                Codes8<T>::expand(pairs(u, x, y, 0), a0, a1);
                                Codes8<T>::expand(pairs(u, x, y, 2), a2, a3);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) M::mma(o[nt][2 * x + y], a0, a1, a2, a3, pb[u][nt][0], pb[u][nt][1]);
                            }
                }
            }
            __syncwarp();                                                // every lane has used what it read
            if (lane == 0) ptx::mbar_arrive(&s_free[warp][slot]);
            if (++slot == C::kStages) {
                slot = 0;
                par ^= 1u;
            }
        }

        // ---- merge: warps, then the CTAs of the cluster
        float *sum = reinterpret_cast<float *>(fifo);                    // [kCols][D]
        __syncwarp();                                                    // the warp's last reads of its FIFO
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int col = 8 * nt + 2 * c + x;
                float v = l[nt][x];
#pragma unroll
                for (int y = 4; y < 32; y <<= 1) v += __shfl_xor_sync(~0u, v, y);
                if (r == 0) {
                    s_m[warp][col] = m[nt][x];
                    s_l[warp][col] = v;
                }
            }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
                for (int x = 0; x < 2; ++x)                              // m-tile mt: columns 64 (mt / 4) + 8 r + 2 (mt % 4) and the next
                    *reinterpret_cast<float2 *>(sum + (8 * nt + 2 * c + x) * D + 64 * (mt / 4) + 8 * r + 2 * (mt % 4)) =
                        make_float2(o[nt][mt][x], o[nt][mt][2 + x]);
    }
    if (failed) {
        p.seqs.raise(VQ_WORD_TIMEOUT);
#pragma unroll 1
        for (int x = 0; x < (1 << 14); ++x) __nanosleep(256);        // tile loads still in flight get time to land
    }
    __syncthreads();
    const auto sum_of = [&](int w) { return reinterpret_cast<float *>(smem + w * C::kWarpBytes); };
    T *out = static_cast<T *>(p.out);
    auto store = [&](int col, int d, float4 v, float den) {
        const float inv = den != 0.f ? 1.f / den : 0.f;
        const int64_t t = t0 + col / p.G, h = hk * p.G + col % p.G;
        *reinterpret_cast<uint2 *>(out + t * p.o_t + h * p.o_h + d) = make_uint2(Pair16<T>::pack(v.x * inv, v.y * inv), Pair16<T>::pack(v.z * inv, v.w * inv));
    };
    for (int x = tid; x < rows * (D / 4); x += C::kThreads) {
        const int col = x / (D / 4), d = x % (D / 4) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) mm = fmaxf(mm, s_m[w][col]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < C::kWarps; ++w) {
            const float a = s_m[w][col] == -INFINITY ? 0.f : ptx::ex2(s_m[w][col] - mm);
            const float4 y = *reinterpret_cast<const float4 *>(sum_of(w) + col * D + d);
            v.x = fmaf(a, y.x, v.x); v.y = fmaf(a, y.y, v.y); v.z = fmaf(a, y.z, v.z); v.w = fmaf(a, y.w, v.w);
            den = fmaf(a, s_l[w][col], den);
        }
        if (nsplit == 1) {
            store(col, d, v, den);
            continue;
        }
        *reinterpret_cast<float4 *>(sum_of(0) + col * D + d) = v;    // only this thread reads or writes these four columns
        if (d == 0) {
            s_cm[col] = mm;
            s_cl[col] = den;
        }
    }
    if (nsplit == 1) return;
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int x = split * C::kThreads + tid; x < rows * (D / 4); x += nsplit * C::kThreads) {
        const int col = x / (D / 4), d = x % (D / 4) * 4;
        // four CTAs at a time, their loads under way together
        float mm = -INFINITY, den = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < nsplit; k0 += 4) {
            float mk[4], lk[4];
            float4 y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int from = min(k0 + k, nsplit - 1);
                mk[k] = *cluster.map_shared_rank(&s_cm[col], from);
                lk[k] = *cluster.map_shared_rank(&s_cl[col], from);
                y[k] = *cluster.map_shared_rank(reinterpret_cast<float4 *>(sum_of(0) + col * D + d), from);
                if (k0 + k >= nsplit) mk[k] = -INFINITY;
            }
            const float top = fmaxf(mm, fmaxf(fmaxf(mk[0], mk[1]), fmaxf(mk[2], mk[3])));
            const float keep = mm == -INFINITY ? 0.f : ptx::ex2(mm - top);
            v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep;
            den *= keep;
            mm = top;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float a = mk[k] == -INFINITY ? 0.f : ptx::ex2(mk[k] - top);
                v.x = fmaf(a, y[k].x, v.x); v.y = fmaf(a, y[k].y, v.y); v.z = fmaf(a, y[k].z, v.z); v.w = fmaf(a, y[k].w, v.w);
                den = fmaf(a, lk[k], den);
            }
        }
        store(col, d, v, den);
    }
    cluster.sync();                                                  // nobody leaves while others read its sums
}

// pool [NP, Hkv, P, D] in boxes of 16 rows x 64 columns of 16 bits, or whole rows of 8 bits
template <bool Q8>
static bool map_rows(CUtensorMap *out, const PagedPool &pool, const PagedAttnParams &p, bool f16)
{
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return false;
    const int P = 1 << p.seqs.log_p, e = Q8 ? 1 : 2;
    const cuuint64_t dim[4] = {static_cast<cuuint64_t>(p.D), static_cast<cuuint64_t>(P), static_cast<cuuint64_t>(p.Hkv), static_cast<cuuint64_t>(p.seqs.NP)};
    // a dimension of one element may come with any stride: give the map one it accepts
    const cuuint64_t str[3] = {static_cast<cuuint64_t>(pool.s_row * e), static_cast<cuuint64_t>((p.Hkv > 1 ? pool.s_head : pool.s_row) * e),
                               static_cast<cuuint64_t>((p.seqs.NP > 1 ? pool.s_page : pool.s_row) * e)};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(Q8 ? p.D : 64), 16, 1, 1}, es[4] = {1, 1, 1, 1};
    return fn(out, Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
              const_cast<void *>(pool.ptr), dim, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              Q8 && p.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool Q8, int D, int NT>
static int launch_few(const PagedAttnParams &p, cudaStream_t stream)
{
    using C = FewCfg<T, Q8, D, NT>;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return VQ_EDEVICE;
    auto kern = paged_few_kernel<T, Q8, D, NT>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return VQ_ELAUNCH;
    const int groups = p.max_q > 1 ? 2 : 1;                          // tokens of one sequence lie in at most two blocks of positions
    const int64_t units = static_cast<int64_t>(p.seqs.S) * groups * p.Hkv;
    int nsplit = 1;
    // As many CTAs of a cluster as the SMs hold at once: a second round would start when the first one ends.  (The second block of positions of a
    // sequence is hardly ever there.)
    while (nsplit < kFewSplit && 2 * nsplit * p.seqs.S * static_cast<int64_t>(p.Hkv) <= C::kCtas * sms) nsplit *= 2;
    if (units * nsplit > 0x7fffffff) return VQ_EUNSUPPORTED;
    constexpr bool f16 = !IsBf16<T>::value;
    CUtensorMap k1, k3, v, cb, vs;
    if (!map_rows<Q8>(&k1, p.k1, p, f16) || !map_rows<Q8>(&k3, p.k3, p, f16) || !map_rows<Q8>(&v, p.v, p, f16)) return VQ_ELAUNCH;
    if (p.cb != nullptr) {
        const uint64_t MK = p.MK, cd[3] = {D, MK, static_cast<uint64_t>(p.Hkv)}, cs[3] = {1, D, MK * D}, vd[3] = {D, MK, static_cast<uint64_t>(p.NS) * p.Hkv};
        if (!make_map(&cb, p.cb, 3, cd, cs, 16, f16) || !make_map(&vs, p.vsum, 3, vd, cs, 16, f16)) return VQ_ELAUNCH;
    } else {
        cb = vs = k1;               // never read
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(nsplit);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // see launch_overlapped
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(units * nsplit));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kTotal;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, k1, k3, v, cb, vs, p, nsplit) == cudaSuccess ? launch_status() : (cudaGetLastError(), VQ_ELAUNCH);
}

template <typename T, bool Q8, int D>
static int launch_few_rows(const PagedAttnParams &p, cudaStream_t stream)
{
    const int rows = p.max_q * p.G;
    return rows <= 8 ? launch_few<T, Q8, D, 1>(p, stream) : rows <= 16 ? launch_few<T, Q8, D, 2>(p, stream) : launch_few<T, Q8, D, 4>(p, stream);
}

template <typename T>
static int launch_few_type(const PagedAttnParams &p, bool q8, cudaStream_t stream)
{
    if (p.D == 64) return q8 ? launch_few_rows<T, true, 64>(p, stream) : launch_few_rows<T, false, 64>(p, stream);
    return q8 ? launch_few_rows<T, true, 128>(p, stream) : launch_few_rows<T, false, 128>(p, stream);
}

int launch_paged_few(const PagedAttnParams &p, int dtype, bool q8, cudaStream_t stream)
{
    return dtype == VQ_F16 ? launch_few_type<__half>(p, q8, stream) : launch_few_type<__nv_bfloat16>(p, q8, stream);
}

}  // namespace vq
