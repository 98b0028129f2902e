// Attention over a paged cache in full precision (fp32 or 8-bit rows), any number of new tokens.
//
// A CTA owns 32 query rows of one kv head - its query heads times tokens of one 128-block of positions - and walks steps of 32 codes or keys with
// one online softmax.  Both products are register tiles on the fp32 pipe, which bounds it (2 * 32 * 32 * D multiply-adds a step): a thread scores 2
// rows x 4 keys, then owns 2 rows x D / 8 columns of the sums - the same two rows, so maximum, denominator and rescaling stay inside
// groups of eight lanes.  The next step's rows are on their way to registers meanwhile.  Where the tiles do not fill the chip, the CTAs
// of a cluster share a tile's steps and merge their sums through distributed shared memory.
// One warp per query row, each lane a key (the first version): 220 us for 178 tokens of 8 heads of 64 over 512 codes and a window of 128;
// this: 47 us.
#include <cooperative_groups.h>

#include "paged_attn.cuh"

namespace vq {

namespace cg = cooperative_groups;

constexpr int kF32Rows = 32, kF32Keys = 32, kF32Threads = 128, kF32Split = 8;

template <int D>
struct F32Cfg {
    static constexpr int kPitch = D + 4;                 // floats per row of q and K: eight lanes that read together ask for different banks
    static constexpr int kTotal = (2 * kF32Rows * kPitch + kF32Keys * kPitch + kF32Keys * D + kF32Rows * (kF32Keys + 4)) * 4;
};

template <typename KV, int D>
__global__ void __launch_bounds__(kF32Threads, 3) paged_f32_kernel(const PagedAttnParams p, int TQ, int GH, int nsplit)
{
    using C = F32Cfg<D>;
    constexpr int NV = D / 16;                           // 16-byte pieces of a row per thread: four threads share a row
    constexpr bool Q8 = sizeof(KV) == 1;
    extern __shared__ __align__(16) float sm[];
    float *s_q = sm, *s_k = s_q + 2 * kF32Rows * C::kPitch, *s_v = s_k + kF32Keys * C::kPitch, *s_p = s_v + kF32Keys * D;
    __shared__ ChunkTile s_tile;
    __shared__ int s_some;
    __shared__ float s_w[kF32Keys], s_m[kF32Rows], s_l[kF32Rows];
    const int tid = threadIdx.x, hk = blockIdx.y, h0 = hk * p.G + blockIdx.z * GH, heads = min(GH, (hk + 1) * p.G - h0);
    const int split = blockIdx.x % nsplit;
    if (tid < 32) {
        ChunkTile t;
        const bool some = chunk_find(p, TQ, blockIdx.x / nsplit, t);
        if (tid == 0) {
            s_some = some;
            s_tile = t;
        }
    }
    __syncthreads();
    if (!s_some) return;                                 // the whole cluster leaves
    const ChunkTile tile = s_tile;
    const int rows = tile.ntok * heads, i0 = tile.pos0, i1 = tile.pos0 + tile.ntok - 1, bd = p.boundary(i0);
    for (int x = tid; x < 2 * kF32Rows * D; x += kF32Threads) {
        const int which = x / (kF32Rows * D), row = x / D % kF32Rows, d = x % D;
        float v = 0.f;
        if (row < rows) {
            const int64_t t = tile.t0 + row / heads, h = h0 + row % heads;
            v = which ? static_cast<const float *>(p.q2)[t * p.q2_t + h * p.q2_h + d] : static_cast<const float *>(p.q1)[t * p.q1_t + h * p.q1_h + d];
        }
        s_q[(which * kF32Rows + row) * C::kPitch + d] = v;
    }
    // steps: codes, raw keys before the exact window, rotated keys
    const int n_far = tile.snap >= 0 ? p.MK / kF32Keys : 0;
    const int old_end = p.rerope ? max(0, i1 - p.W) : 0, n_old = old_end > bd ? (old_end - bd + kF32Keys - 1) / kF32Keys : 0;
    const int near0 = (p.rerope ? max(0, i0 - p.W) : bd) / kF32Keys * kF32Keys, n_near = (i1 - near0) / kF32Keys + 1;
    const int total = n_far + n_old + n_near;
    const int64_t far_base = (static_cast<int64_t>(max(tile.snap, 0)) * p.Hkv + hk) * p.MK;
    const int page_mask = (1 << p.seqs.log_p) - 1;
    auto first_key = [&](int step) { return step < n_far + n_old ? bd + (step - n_far) * kF32Keys : near0 + (step - n_far - n_old) * kF32Keys; };

    // ---- a step's rows: row tid / 4, pieces tid % 4, + 4, ...
    const int lrow = tid >> 2, lp = tid & 3;
    float4 rk[NV], rv[NV];
    float rw = 0.f;                                      // count of a code; 0: a row that is not there
    auto fetch = [&](int step) {
        rw = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) rk[j] = rv[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (step >= total) return;
        if (step < n_far) {
            const int r = step * kF32Keys + lrow;
            const float4 *k = reinterpret_cast<const float4 *>(static_cast<const float *>(p.cb) + (static_cast<int64_t>(hk) * p.MK + r) * D) + lp;
            const float4 *v = reinterpret_cast<const float4 *>(static_cast<const float *>(p.vsum) + (far_base + r) * D) + lp;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                rk[j] = __ldg(k + 4 * j);
                rv[j] = __ldg(v + 4 * j);
            }
            rw = __ldg(p.cnt + far_base + r);
            return;
        }
        const int key = first_key(step) + lrow;
        const int page = key <= i1 ? p.seqs.page(tile.s, key >> p.seqs.log_p) : -1, pr = key & page_mask;
        if (page < 0) return;
        rw = 1.f;
        const bool old = step < n_far + n_old;
        const PagedPool &kp = old ? p.k3 : p.k1;
        const KV *k = static_cast<const KV *>(kp.ptr) + kp.row(page, hk, pr) + 4 * lp;
        const KV *v = static_cast<const KV *>(p.v.ptr) + p.v.row(page, hk, pr) + 4 * lp;
        if constexpr (Q8) {
            float ks = __ldg(kp.scale + kp.scale_at(page, hk, pr)), vs = __ldg(p.v.scale + p.v.scale_at(page, hk, pr));
            if (!(fabsf(vs) < INFINITY)) {                   // a value row that is not finite: its score says so to the tokens that see it
                ks = __int_as_float(0x7fffffff);
                vs = 0.f;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const char4 a = *reinterpret_cast<const char4 *>(k + 16 * j), b = *reinterpret_cast<const char4 *>(v + 16 * j);
                rk[j] = make_float4(dequant(a.x, ks), dequant(a.y, ks), dequant(a.z, ks), dequant(a.w, ks));
                rv[j] = make_float4(dequant(b.x, vs), dequant(b.y, vs), dequant(b.z, vs), dequant(b.w, vs));
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                rk[j] = __ldg(reinterpret_cast<const float4 *>(k + 16 * j));
                rv[j] = __ldg(reinterpret_cast<const float4 *>(v + 16 * j));
            }
        }
    };

    const int ty = tid >> 3, tx = tid & 7, r0 = 2 * ty;  // rows r0, r0 + 1
    float o[2][D / 8], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int d = 0; d < D / 8; ++d) o[a][d] = 0.f;
    fetch(split);
    for (int step = split; step < total; step += nsplit) {
        __syncthreads();                                 // q is there; the step before has been used
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            *reinterpret_cast<float4 *>(s_k + lrow * C::kPitch + 4 * lp + 16 * j) = rk[j];
            *reinterpret_cast<float4 *>(s_v + lrow * D + 4 * lp + 16 * j) = rv[j];
        }
        if (lp == 0) s_w[lrow] = rw;
        fetch(step + nsplit);
        __syncthreads();
        const bool far = step < n_far, old = !far && step < n_far + n_old;
        // ---- scores of rows r0, r0 + 1 and keys tx, 8 + tx, ...
        const float *q = s_q + ((far || old ? kF32Rows : 0) + r0) * C::kPitch;
        float s[2][4], s2[2][4];                         // two partial sums each: shorter chains of roundings
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[a][x] = s2[a][x] = 0.f;
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            const float4 qa = *reinterpret_cast<const float4 *>(q + d), qb = *reinterpret_cast<const float4 *>(q + C::kPitch + d);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float4 k = *reinterpret_cast<const float4 *>(s_k + (tx + 8 * x) * C::kPitch + d);
                s[0][x] = fmaf(qa.z, k.z, fmaf(qa.x, k.x, s[0][x]));
                s2[0][x] = fmaf(qa.w, k.w, fmaf(qa.y, k.y, s2[0][x]));
                s[1][x] = fmaf(qb.z, k.z, fmaf(qb.x, k.x, s[1][x]));
                s2[1][x] = fmaf(qb.w, k.w, fmaf(qb.y, k.y, s2[1][x]));
            }
        }
        const int key0 = first_key(step);
        float w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = s_w[tx + 8 * x];
        float kept[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int i = i0 + (r0 + a) / heads;
            const int hi = old ? i - p.W - 1 : i, lo = old || !p.rerope ? bd : i - p.W;
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int j = key0 + tx + 8 * x;
                s[a][x] += s2[a][x];
                if (!(w[x] > 0.f) || (!far && (j < lo || j > hi))) s[a][x] = -INFINITY;
                mx = fmaxf(mx, s[a][x]);
            }
#pragma unroll
            for (int y = 1; y < 8; y <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, y));
            const float old_m = m[a];
            m[a] = fmaxf(old_m, mx * p.scale_log2);
            const float ref = m[a] == -INFINITY ? 0.f : m[a], keep = old_m == -INFINITY ? 0.f : exp2f(old_m - ref);
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float e = exp2f(fmaf(s[a][x], p.scale_log2, -ref));   // one rounding, of the difference
                sum = fmaf(e, w[x] > 0.f ? w[x] : 0.f, sum);
                s_p[(r0 + a) * (kF32Keys + 4) + tx + 8 * x] = e;
            }
            l[a] = fmaf(l[a], keep, sum);
            kept[a] = keep;
        }
        __syncwarp();                                    // a warp's weights are used by the warp alone
        // ---- sums: rows r0, r0 + 1, columns 4 tx + 32 y
        // A step's sums by themselves, then added to what was kept: in one chain over thousands of keys every addition rounds to the long
        // sum's last bit (1.2e-6 of the result over a window of 4096, 3.4e-7 this way, for 3% of the time).
        const float *pa = s_p + r0 * (kF32Keys + 4), *pb = pa + kF32Keys + 4;
        float t[2][D / 8];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int d = 0; d < D / 8; ++d) t[a][d] = 0.f;
#pragma unroll 2
        for (int j = 0; j < kF32Keys; j += 4) {
            const float4 a4 = *reinterpret_cast<const float4 *>(pa + j), b4 = *reinterpret_cast<const float4 *>(pb + j);
            const float wa[4] = {a4.x, a4.y, a4.z, a4.w}, wb[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int y = 0; y < D / 32; ++y) {
                    const float4 v = *reinterpret_cast<const float4 *>(s_v + (j + x) * D + 4 * tx + 32 * y);
                    t[0][4 * y] = fmaf(wa[x], v.x, t[0][4 * y]); t[0][4 * y + 1] = fmaf(wa[x], v.y, t[0][4 * y + 1]);
                    t[0][4 * y + 2] = fmaf(wa[x], v.z, t[0][4 * y + 2]); t[0][4 * y + 3] = fmaf(wa[x], v.w, t[0][4 * y + 3]);
                    t[1][4 * y] = fmaf(wb[x], v.x, t[1][4 * y]); t[1][4 * y + 1] = fmaf(wb[x], v.y, t[1][4 * y + 1]);
                    t[1][4 * y + 2] = fmaf(wb[x], v.z, t[1][4 * y + 2]); t[1][4 * y + 3] = fmaf(wb[x], v.w, t[1][4 * y + 3]);
                }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int d = 0; d < D / 8; ++d) o[a][d] = fmaf(o[a][d], kept[a], t[a][d]);
    }
    // ---- merge
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int y = 1; y < 8; y <<= 1) l[a] += __shfl_xor_sync(~0u, l[a], y);
    auto store = [&](int row, int d, float4 v, float den) {
        const float inv = den != 0.f ? 1.f / den : 0.f;
        const int64_t t = tile.t0 + row / heads, h = h0 + row % heads;
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + t * p.o_t + h * p.o_h + d) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    };
    if (nsplit == 1) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
            if (r0 + a < rows)
#pragma unroll
                for (int y = 0; y < D / 32; ++y)
                    store(r0 + a, 4 * tx + 32 * y, make_float4(o[a][4 * y], o[a][4 * y + 1], o[a][4 * y + 2], o[a][4 * y + 3]), l[a]);
        return;
    }
    __syncthreads();
    float *s_o = s_q;                                    // [rows][D]: the queries have been used
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
        for (int y = 0; y < D / 32; ++y)
            *reinterpret_cast<float4 *>(s_o + (r0 + a) * D + 4 * tx + 32 * y) = make_float4(o[a][4 * y], o[a][4 * y + 1], o[a][4 * y + 2], o[a][4 * y + 3]);
        if (tx == 0) {
            s_m[r0 + a] = m[a];
            s_l[r0 + a] = l[a];
        }
    }
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int x = split * kF32Threads + tid; x < rows * (D / 4); x += nsplit * kF32Threads) {
        const int row = x / (D / 4), d = x % (D / 4) * 4;
        float mk[kF32Split], lk[kF32Split], top = -INFINITY, den = 0.f;
        float4 y[kF32Split], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kF32Split; ++k) {
            const int from = min(k, nsplit - 1);
            mk[k] = k < nsplit ? *cluster.map_shared_rank(&s_m[row], from) : -INFINITY;
            lk[k] = *cluster.map_shared_rank(&s_l[row], from);
            y[k] = *cluster.map_shared_rank(reinterpret_cast<float4 *>(s_o + row * D + d), from);
            top = fmaxf(top, mk[k]);
        }
#pragma unroll
        for (int k = 0; k < kF32Split; ++k) {
            if (k >= nsplit) break;
            // without a maximum there are no weights, or none that is a number
            const float a = mk[k] == -INFINITY ? (lk[k] != lk[k] ? 1.f : 0.f) : exp2f(mk[k] - top);
            v.x = fmaf(a, y[k].x, v.x); v.y = fmaf(a, y[k].y, v.y); v.z = fmaf(a, y[k].z, v.z); v.w = fmaf(a, y[k].w, v.w);
            den = fmaf(a, lk[k], den);
        }
        store(row, d, v, den);
    }
    cluster.sync();                                      // nobody leaves while others read its sums
}

template <typename KV, int D>
static int launch_f32(const PagedAttnParams &p, cudaStream_t stream)
{
    using C = F32Cfg<D>;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return VQ_EDEVICE;
    auto kern = paged_f32_kernel<KV, D>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal) != cudaSuccess) return VQ_ELAUNCH;
    const int GH = p.G < kF32Rows ? p.G : kF32Rows, TQ = kF32Rows / GH, hz = (p.G + GH - 1) / GH;
    const int64_t tiles = chunk_tiles(p.seqs, TQ), ctas = tiles * p.Hkv * hz;
    int nsplit = 1;
    while (nsplit < kF32Split && 2 * nsplit * ctas <= 3 * sms) nsplit *= 2;
    if (tiles * nsplit > 0x7fffffff) return VQ_EUNSUPPORTED;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(nsplit);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * nsplit), static_cast<unsigned>(p.Hkv), static_cast<unsigned>(hz));
    cfg.blockDim = dim3(kF32Threads);
    cfg.dynamicSmemBytes = C::kTotal;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p, TQ, GH, nsplit) == cudaSuccess ? launch_status() : (cudaGetLastError(), VQ_ELAUNCH);
}

int launch_paged_f32(const PagedAttnParams &p, bool q8, cudaStream_t stream)
{
    if (p.D == 64) return q8 ? launch_f32<int8_t, 64>(p, stream) : launch_f32<float, 64>(p, stream);
    return q8 ? launch_f32<int8_t, 128>(p, stream) : launch_f32<float, 128>(p, stream);
}

}  // namespace vq
