// Attention over a paged cache for few new tokens per sequence (one token of a decode, a handful of drafted ones): at most 32 query rows -
// tokens times query heads - share a kv head's keys.
//
// Bound by HBM: 4 D operations per key and row against 4 D (2 D) bytes per key.  So the work is organised around the stream of rows, and the
// matrix product only has to keep out of its way: mma.sync with the KEYS on the M axis (16 per instruction) and 8 query rows on N, for
// which a tile of 128 rows of tcgen05 would be nearly empty.  A warp takes steps of 16 keys (32 of 8-bit rows) and keeps its own online
// softmax: no barrier in the loop.
//   - Both products may permute their reduction index: a thread reads 16 contiguous bytes of a key row, which hold its operands of
//     several k-steps, and q is read in the same order.  Values enter as V^T (D on M): pairs of keys are interleaved by byte permutes.
//     So every thread copies exactly the bytes it will use (cp.async, a private FIFO in shared memory): no shared layout, no ldmatrix, not
//     even a warp barrier between copy and use.
//   - S^T (keys x rows) becomes the B operand of the second product by movmatrix, 8 x 8 at a time.
//   - 8-bit codes become 16-bit floats exactly (byte permutes and one subtraction); a key's scale multiplies its score, a value's scale its
//     weight.
//   - Counts multiply the weights of codes in the denominator; codes without members are excluded.
// One unit = (sequence, block of positions, kv head); its steps are dealt out to the warps of a cluster of 1 - 8 CTAs, which merge their
// partial sums through distributed shared memory: no workspace, no second launch, the same order of additions every time.
#include <cooperative_groups.h>

#include "codes8.cuh"
#include "paged_attn.cuh"
#include "tc_ptx.cuh"

namespace vq {

namespace cg = cooperative_groups;

constexpr int kFewWarps = 4;
constexpr int kFewStages = 3;
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
// copies N bytes, or zeros when !some
template <int N>
__device__ __forceinline__ void cp_async(void *dst, const void *src, bool some)
{
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(some ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(ptx::smem_u32(dst)), "l"(src), "n"(N), "r"(some ? N : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, bool Q8, int D, int NT>
struct FewCfg {
    static constexpr int kCols = 8 * NT;                         // query rows, padded
    static constexpr int KC = D / 32, VC = D / 64;               // 16-byte pieces of a 16-bit key / value row per thread
    static constexpr int kSlots16 = 2 * KC + 4 * VC;             // 16-byte slots per thread: 16 keys of 16-bit rows
    static constexpr int kSlots8 = 2 * (2 * VC + 4);             // 32 keys of 8-bit rows
    static constexpr int kSlots = Q8 && kSlots8 > kSlots16 ? kSlots8 : kSlots16;
    static constexpr int kStage = kSlots * 32 * 16;              // bytes of a stage: 16 keys, or 32 of 8-bit rows
    static constexpr int kScal = (Q8 ? 8 : 2) * 32 * 4;          // counts, or scales of keys and values
    static constexpr int kWarpBytes = kFewStages * (kStage + kScal);
    static constexpr int kQ = 2 * kCols * D * 2;                 // q1 and q2 rows
    static constexpr int kPages = Q8 ? 64 : 512;                 // page table entries kept in shared memory (the rest is read where it is
                                                                 // needed): 8-bit rows leave no more if two CTAs are to share an SM
    static constexpr int kTotal = kFewWarps * kWarpBytes + kQ + kPages * 4;
    static_assert(kCols * D * 4 <= kFewStages * kStage, "a warp's sums fit into its FIFO");
    static constexpr int MT = D / 16;
};

struct FewSteps {
    int n_far, n_old, n_near;       // steps of codes, of raw keys before the exact window, of rotated keys
    int old0, near0;                // first key of the latter two (multiples of 16)
};

template <typename T, bool Q8, int D, int NT>
__global__ void __launch_bounds__(kFewWarps * 32) paged_few_kernel(const PagedAttnParams p, int groups, int nsplit)
{
    using C = FewCfg<T, Q8, D, NT>;
    using M = Mma16816<T>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_m[kFewWarps][C::kCols], s_l[kFewWarps][C::kCols];
    __shared__ float s_cm[C::kCols], s_cl[C::kCols];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r = lane >> 2, c = lane & 3;
    uint8_t *fifo = smem + warp * C::kWarpBytes;
    T *s_q = reinterpret_cast<T *>(smem + kFewWarps * C::kWarpBytes);        // [2][kCols][D]
    int *s_page = reinterpret_cast<int *>(smem + kFewWarps * C::kWarpBytes + C::kQ);

    const int split = blockIdx.x % nsplit;
    int unit = blockIdx.x / nsplit;
    const int hk = unit % p.Hkv;
    unit /= p.Hkv;
    const int grp = unit % groups, s = unit / groups;
    int t0, q, n;
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
    const int bd = p.boundary(i0), snap = p.snapshot(s, bd);
    FewSteps st;
    constexpr bool kHalf = Q8 && !IsBf16<T>::value;
    constexpr int KEYS = Q8 ? 32 : 16;                               // keys per step of window rows
    st.n_far = snap >= 0 ? p.MK / 16 : 0;
    st.old0 = bd;
    const int old_end = p.rerope ? max(0, i1 - p.W) : 0;             // raw keys: [bd, old_end)
    st.n_old = old_end > bd ? (old_end - bd + KEYS - 1) / KEYS : 0;
    st.near0 = (p.rerope ? max(0, i0 - p.W) : bd) & ~15;
    st.n_near = (i1 - st.near0) / KEYS + 1;
    const int total = st.n_far + st.n_old + st.n_near;
    const int col0 = bd >> p.seqs.log_p, cols = (i1 >> p.seqs.log_p) - col0 + 1;

    for (int x = tid; x < min(cols, C::kPages); x += kFewWarps * 32) s_page[x] = p.seqs.page(s, col0 + x);
    for (int x = tid; x < 2 * C::kCols * D / 8; x += kFewWarps * 32) {
        const int which = x / (C::kCols * D / 8), row = x / (D / 8) % C::kCols, d = x % (D / 8) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row < rows) {
            const int64_t t = t0 + row / p.G, h = hk * p.G + row % p.G;
            const T *src = which ? static_cast<const T *>(p.q2) + t * p.q2_t + h * p.q2_h : static_cast<const T *>(p.q1) + t * p.q1_t + h * p.q1_h;
            v = *reinterpret_cast<const uint4 *>(src + d);
        }
        reinterpret_cast<uint4 *>(s_q)[x] = v;
    }
    __syncthreads();

    const int64_t far_base = (static_cast<int64_t>(snap < 0 ? 0 : snap) * p.Hkv + hk) * p.MK;
    const int page_mask = (1 << p.seqs.log_p) - 1;
    auto page_of = [&](int j) {
        const int x = (j >> p.seqs.log_p) - col0;
        return x < C::kPages ? s_page[x] : p.seqs.page(s, x + col0);
    };
    // ---- the thread's share of a step, into stage `slot`
    auto fill = [&](int step, int slot) {
        uint8_t *dst = fifo + slot * C::kStage;
        float *sc = reinterpret_cast<float *>(fifo + kFewStages * C::kStage + slot * C::kScal);
        if (step < st.n_far) {
            const int r0 = step * 16;
            const T *kb = static_cast<const T *>(p.cb) + (static_cast<int64_t>(hk) * p.MK + r0) * D;
            const T *vb = static_cast<const T *>(p.vsum) + (far_base + r0) * D;
            int x = 0;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int j = 0; j < C::KC; ++j, ++x) cp_async<16>(dst + (x * 32 + lane) * 16, kb + (r + 8 * a) * D + 32 * j + 8 * c, true);
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int j = 0; j < C::VC; ++j, ++x)
                    cp_async<16>(dst + (x * 32 + lane) * 16, vb + (2 * c + (a & 1) + 8 * (a >> 1)) * D + 64 * j + 8 * r, true);
#pragma unroll
            for (int a = 0; a < 2; ++a) cp_async<4>(sc + a * 32 + lane, p.cnt + far_base + r0 + r + 8 * a, true);
            return;
        }
        const bool old = step < st.n_far + st.n_old;
        const int key0 = old ? st.old0 + (step - st.n_far) * KEYS : st.near0 + (step - st.n_far - st.n_old) * KEYS;
        const PagedPool &kp = old ? p.k3 : p.k1;
        int x = 0;
#pragma unroll
        for (int sub = 0; sub < KEYS / 16; ++sub) {
            const int j0 = key0 + 16 * sub;
            const int pg = j0 <= i1 ? page_of(j0) : -1;               // none: zeros, whose keys are masked (or reported)
            const bool have = pg >= 0;
            const int pr = j0 & page_mask, page = have ? pg : 0;
            if constexpr (!Q8) {
                const T *kb = static_cast<const T *>(kp.ptr) + kp.row(page, hk, pr), *vb = static_cast<const T *>(p.v.ptr) + p.v.row(page, hk, pr);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int j = 0; j < C::KC; ++j, ++x) cp_async<16>(dst + (x * 32 + lane) * 16, kb + (r + 8 * a) * kp.s_row + 32 * j + 8 * c, have);
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const int key = 2 * c + (a & 1) + 8 * (a >> 1);
#pragma unroll
                    for (int j = 0; j < C::VC; ++j, ++x)              // behind the sequence's end a page may hold anything: zeros instead
                        cp_async<16>(dst + (x * 32 + lane) * 16, vb + key * p.v.s_row + 64 * j + 8 * r, have && j0 + key < n);
                }
            } else {
                const int8_t *kb = static_cast<const int8_t *>(kp.ptr) + kp.row(page, hk, pr), *vb = static_cast<const int8_t *>(p.v.ptr) + p.v.row(page, hk, pr);
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int j = 0; j < D / 64; ++j, ++x) cp_async<16>(dst + (x * 32 + lane) * 16, kb + (r + 8 * a) * kp.s_row + 64 * j + 16 * c, have);
#pragma unroll
                for (int a = 0; a < 4; ++a, ++x) {
                    const int key = 2 * c + (a & 1) + 8 * (a >> 1);
#pragma unroll
                    for (int j = 0; j < C::VC; ++j) cp_async<8>(dst + (x * 32 + lane) * 16 + 8 * j, vb + key * p.v.s_row + 64 * j + 8 * r, have);
                }
                const float *ks = kp.scale + kp.scale_at(page, hk, pr), *vs = p.v.scale + p.v.scale_at(page, hk, pr);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const bool in = have && j0 + r + 8 * a < n;
                    cp_async<4>(sc + (4 * sub + a) * 32 + lane, ks + (r + 8 * a) * kp.c_row, in);
                    cp_async<4>(sc + (4 * sub + 2 + a) * 32 + lane, vs + (r + 8 * a) * p.v.c_row, in);
                }
            }
        }
    };

    float o[NT][C::MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[nt][mt][x] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
    }
    uint32_t qf[NT][D / 8];

    const int stride = nsplit * kFewWarps, first = split * kFewWarps + warp;
#pragma unroll
    for (int x = 0; x < kFewStages - 1; ++x) {
        if (first + x * stride < total) fill(first + x * stride, x);
        cp_commit();
    }
    // positions of the thread's columns
    int pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) pos[nt][x] = i0 + (8 * nt + 2 * c + x) / p.G;

    // sc: scores of keys r and r + 8 (c0 c1 | c2 c3) in log2 units, -inf where excluded -> weights; w: denominator weights of the two keys,
    // f: factors of their value rows.  Raises the references, adds to l, returns the packed weights as B operands.
    auto softmax = [&](float (&sc)[NT][4], float w0, float w1, float f0, float f1, uint32_t (&pb)[NT][2]) {
        bool above = false;
        float mx[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                mx[nt][x] = fmaxf(sc[nt][x], sc[nt][2 + x]);
                above |= mx[nt][x] > m[nt][x] + kFewLazy || (m[nt][x] == -INFINITY && mx[nt][x] > -INFINITY);
            }
        if (__any_sync(~0u, above)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float v = mx[nt][x];
#pragma unroll
                    for (int y = 4; y < 32; y <<= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, y));
                    if (v > m[nt][x]) {
                        const float a = m[nt][x] == -INFINITY ? 0.f : ptx::ex2(m[nt][x] - v);
                        m[nt][x] = v;
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
            const float p0 = ptx::ex2(sc[nt][0] - ma), p1 = ptx::ex2(sc[nt][1] - mb), p2 = ptx::ex2(sc[nt][2] - ma), p3 = ptx::ex2(sc[nt][3] - mb);
            l[nt][0] += p0 * w0 + p2 * w1;
            l[nt][1] += p1 * w0 + p3 * w1;
            pb[nt][0] = movmatrix(Pair16<T>::pack(p0 * f0, p1 * f0));
            pb[nt][1] = movmatrix(Pair16<T>::pack(p2 * f1, p3 * f1));
        }
    };

    int phase = -1, slot = 0;
    for (int step = first; step < total; step += stride) {
        {
            const int next = step + (kFewStages - 1) * stride;
            int ns = slot + kFewStages - 1;
            if (ns >= kFewStages) ns -= kFewStages;
            if (next < total) fill(next, ns);
            cp_commit();
        }
        const bool far = step < st.n_far, old = !far && step < st.n_far + st.n_old;
        const int ph = far ? 0 : old ? 1 : 2;
        if (ph != phase) {                                           // q in the order of this phase's key rows
            phase = ph;
            const T *src = s_q + ((far || old) ? C::kCols * D : 0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const T *row = src + (8 * nt + r) * D;
                if (far || !Q8) {
#pragma unroll
                    for (int j = 0; j < C::KC; ++j) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(row + 32 * j + 8 * c);
                        qf[nt][4 * j] = v.x; qf[nt][4 * j + 1] = v.y; qf[nt][4 * j + 2] = v.z; qf[nt][4 * j + 3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < C::KC; ++j) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(row + 64 * (j / 2) + 16 * c + 8 * (j % 2));
                        qf[nt][4 * j] = v.x; qf[nt][4 * j + 1] = v.y; qf[nt][4 * j + 2] = v.z; qf[nt][4 * j + 3] = v.w;
                    }
                }
            }
        }
        cp_wait<kFewStages - 1>();
        const uint8_t *stg = fifo + slot * C::kStage + lane * 16;
        const float *scal = reinterpret_cast<const float *>(fifo + kFewStages * C::kStage + slot * C::kScal) + lane;
        if (++slot == kFewStages) slot = 0;
        const int subs = far || !Q8 ? 1 : 2;
#pragma unroll 1
        for (int sub = 0; sub < subs; ++sub) {
            // ---- S^T = K Q^T
            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[nt][x] = 0.f;
            float w0 = 1.f, w1 = 1.f, f0 = 1.f, f1 = 1.f, k0 = p.scale_log2, k1 = p.scale_log2, e0 = 1.f, e1 = 1.f;
            const uint8_t *kst = stg;
            if (far || !Q8) {
#pragma unroll
                for (int j = 0; j < C::KC; ++j) {
                    const uint4 a = *reinterpret_cast<const uint4 *>(kst + j * 512), b = *reinterpret_cast<const uint4 *>(kst + (C::KC + j) * 512);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        M::mma(sc[nt], a.x, b.x, a.y, b.y, qf[nt][4 * j], qf[nt][4 * j + 1]);
                        M::mma(sc[nt], a.z, b.z, a.w, b.w, qf[nt][4 * j + 2], qf[nt][4 * j + 3]);
                    }
                }
                if (far) {
                    w0 = scal[0];
                    w1 = scal[32];
                }
            } else {
                kst += sub * (2 * (D / 64) + 4) * 512;
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    const uint4 a4 = *reinterpret_cast<const uint4 *>(kst + j * 512), b4 = *reinterpret_cast<const uint4 *>(kst + (D / 64 + j) * 512);
                    const uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t al, ah, bl, bh;
                        Codes8<T>::expand(a[w], al, ah);
                        Codes8<T>::expand(b[w], bl, bh);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) M::mma(sc[nt], al, bl, ah, bh, qf[nt][8 * j + 2 * w], qf[nt][8 * j + 2 * w + 1]);
                    }
                }
                const float *s4 = scal + 4 * sub * 32;
                k0 *= s4[0];
                k1 *= s4[32];
                f0 = s4[64];
                f1 = s4[96];
                if constexpr (kHalf) {
                    f0 = half_weight_factor(f0, e0);
                    f1 = half_weight_factor(f1, e1);
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                sc[nt][0] *= k0; sc[nt][1] *= k0; sc[nt][2] *= k1; sc[nt][3] *= k1;
            }
            // ---- excluded keys
            if (far) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (!(w0 > 0.f)) sc[nt][0] = sc[nt][1] = -INFINITY;
                    if (!(w1 > 0.f)) sc[nt][2] = sc[nt][3] = -INFINITY;
                }
            } else {
                const int j0 = (old ? st.old0 + (step - st.n_far) * KEYS : st.near0 + (step - st.n_far - st.n_old) * KEYS) + 16 * sub;
                // keys every row of the group sees: raw ones below i0 - W, rotated ones in [i1 - W, i0]
                const bool all = old ? j0 + 15 < i0 - p.W : j0 + 15 <= i0 && (!p.rerope || j0 >= i1 - p.W);
                if (!all) {
                    const int ja = j0 + r, jb = ja + 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int i = pos[nt][x], hi = old ? i - p.W - 1 : i, lo = old || !p.rerope ? bd : i - p.W;
                            if (ja < lo || ja > hi || ja >= n) sc[nt][x] = -INFINITY;
                            if (jb < lo || jb > hi || jb >= n) sc[nt][2 + x] = -INFINITY;
                        }
                }
            }
            uint32_t pb[NT][2];
            softmax(sc, w0, w1, f0, f1, pb);
            // ---- O^T += V^T P^T
            if (far || !Q8) {
                const uint8_t *vst = stg + 2 * C::KC * 512;
#pragma unroll
                for (int j = 0; j < C::VC; ++j) {
                    uint4 v4[4];
#pragma unroll
                    for (int a = 0; a < 4; ++a) v4[a] = *reinterpret_cast<const uint4 *>(vst + (a * C::VC + j) * 512);
                    const uint32_t v0[4] = {v4[0].x, v4[0].y, v4[0].z, v4[0].w}, v1[4] = {v4[1].x, v4[1].y, v4[1].z, v4[1].w};
                    const uint32_t v2[4] = {v4[2].x, v4[2].y, v4[2].z, v4[2].w}, v3[4] = {v4[3].x, v4[3].y, v4[3].z, v4[3].w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = __byte_perm(v0[w], v1[w], 0x5410), a1 = __byte_perm(v0[w], v1[w], 0x7632);
                        const uint32_t a2 = __byte_perm(v2[w], v3[w], 0x5410), a3 = __byte_perm(v2[w], v3[w], 0x7632);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) M::mma(o[nt][4 * j + w], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                    }
                }
            } else {
                const uint8_t *vst = stg + (sub * (2 * (D / 64) + 4) + 2 * (D / 64)) * 512;
                uint32_t v[4][D / 32];
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    if constexpr (D == 128) {
                        const uint4 x = *reinterpret_cast<const uint4 *>(vst + a * 512);
                        v[a][0] = x.x; v[a][1] = x.y; v[a][2] = x.z; v[a][3] = x.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2 *>(vst + a * 512);
                        v[a][0] = x.x; v[a][1] = x.y;
                    }
                }
                __half2 pa, pc;                                      // the powers of two that go with this thread's pairs of keys
                if constexpr (kHalf) {
                    pa = __floats2half2_rn(__shfl_sync(~0u, e0, 8 * c), __shfl_sync(~0u, e0, 8 * c + 4));
                    pc = __floats2half2_rn(__shfl_sync(~0u, e1, 8 * c), __shfl_sync(~0u, e1, 8 * c + 4));
                }
#pragma unroll
                for (int w = 0; w < D / 32; ++w)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {           // bytes 0, 1 and 2, 3 of the word: m-tiles 2 w, 2 w + 1
                        uint32_t a0, a1, a2, a3;
                        const uint32_t u = __byte_perm(v[0][w], v[1][w], half ? 0x7362 : 0x5140), x = __byte_perm(v[2][w], v[3][w], half ? 0x7362 : 0x5140);
                        if constexpr (kHalf) {
                            Codes8<T>::expand_scaled(u, pa, a0, a1);
                            Codes8<T>::expand_scaled(x, pc, a2, a3);
                        } else {
                            Codes8<T>::expand(u, a0, a1);
                            Codes8<T>::expand(x, a2, a3);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) M::mma(o[nt][2 * w + half], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                    }
            }
        }
    }
    cp_wait<0>();

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
    __syncthreads();
    const auto sum_of = [&](int w) { return reinterpret_cast<float *>(smem + w * C::kWarpBytes); };
    T *out = static_cast<T *>(p.out);
    auto store = [&](int col, int d, float4 v, float den) {
        const float inv = den != 0.f ? 1.f / den : 0.f;
        const int64_t t = t0 + col / p.G, h = hk * p.G + col % p.G;
        *reinterpret_cast<uint2 *>(out + t * p.o_t + h * p.o_h + d) = make_uint2(Pair16<T>::pack(v.x * inv, v.y * inv), Pair16<T>::pack(v.z * inv, v.w * inv));
    };
    for (int x = tid; x < rows * (D / 4); x += kFewWarps * 32) {
        const int col = x / (D / 4), d = x % (D / 4) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) mm = fmaxf(mm, s_m[w][col]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
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
    for (int x = split * (kFewWarps * 32) + tid; x < rows * (D / 4); x += nsplit * (kFewWarps * 32)) {
        const int col = x / (D / 4), d = x % (D / 4) * 4;
        float mm = -INFINITY;
        for (int k = 0; k < nsplit; ++k) mm = fmaxf(mm, *cluster.map_shared_rank(&s_cm[col], k));
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
        for (int k = 0; k < nsplit; ++k) {
            const float mk = *cluster.map_shared_rank(&s_cm[col], k), a = mk == -INFINITY ? 0.f : ptx::ex2(mk - mm);
            const float4 y = *cluster.map_shared_rank(reinterpret_cast<float4 *>(sum_of(0) + col * D + d), k);
            v.x = fmaf(a, y.x, v.x); v.y = fmaf(a, y.y, v.y); v.z = fmaf(a, y.z, v.z); v.w = fmaf(a, y.w, v.w);
            den = fmaf(a, *cluster.map_shared_rank(&s_cl[col], k), den);
        }
        store(col, d, v, den);
    }
    cluster.sync();                                                  // nobody leaves while others read its sums
}

template <typename T, bool Q8, int D, int NT>
static int launch_few(const PagedAttnParams &p, cudaStream_t stream)
{
    using C = FewCfg<T, Q8, D, NT>;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return VQ_EDEVICE;
    auto kern = paged_few_kernel<T, Q8, D, NT>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal) != cudaSuccess) return VQ_ELAUNCH;
    const int groups = p.max_q > 1 ? 2 : 1;                          // tokens of one sequence lie in at most two blocks of positions
    const int64_t units = static_cast<int64_t>(p.seqs.S) * groups * p.Hkv;
    int nsplit = 1;
    while (nsplit < 8 && units * nsplit < 2 * sms) nsplit *= 2;
    if (units * nsplit > 0x7fffffff) return VQ_EUNSUPPORTED;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(nsplit);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(units * nsplit));
    cfg.blockDim = dim3(kFewWarps * 32);
    cfg.dynamicSmemBytes = C::kTotal;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p, groups, nsplit) == cudaSuccess ? launch_status() : (cudaGetLastError(), VQ_ELAUNCH);
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
