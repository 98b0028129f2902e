// Attention of new tokens over a paged cache: the entry point.  16-bit activations: paged_few.cu (few rows per sequence and kv head) and
// paged_chunk.cu; fp32: paged_f32.cu.
#include "paged_attn.cuh"

namespace vq {

// The line between the forms, in us, few / chunk, 8 kv heads, MK1024, W1024.  16 rows: 8 sequences 18 / 34, 32 sequences 46 / 75; 32 rows: 8
// sequences 31 / 35 (8 bits 39 / 59; D = 64 23 / 33), 32 sequences 94 / 77 (8 bits 125 / 127; D = 64 68 / 72): more than 16 rows of
// 16-bit caches with D = 128 go to the chunk form once the pairs of sequences and heads fill the chip.
static bool few_form(int64_t max_q, int64_t G, int64_t D, bool q8, int64_t units, int sms)
{
    const int64_t rows = max_q * G;
    return rows <= 16 || (rows <= kFewRows && (q8 || D == 64 || units <= sms));
}

// three pools of blocks as 16-bit floats, a factor per row
static size_t workspace_bytes(int64_t blocks, int64_t Hkv, int64_t D) { return static_cast<size_t>(3 * blocks * Hkv * kBlock * (D * 2 + 4)); }

}  // namespace vq

extern "C" size_t vqattn_paged_attention_workspace_bytes(int64_t S, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t max_q,
                                                         int32_t pool_dtype, int32_t act_dtype)
{
    using namespace vq;
    if (pool_dtype != VQ_I8 || !is_16bit(act_dtype) || S <= 0 || T <= 0 || Hkv <= 0 || Hq < Hkv || (D != 64 && D != 128) || window <= 0 || max_q <= 0) return 0;
    if (S > (1 << 20) || T > 0x7fffffff || window > 0x40000000 || Hkv > 65535) return 0;
    const int64_t G = Hq / Hkv, q = max_q < T ? max_q : T;
    if (few_form(q, G, D, true, S * Hkv, 0) || !convert_first(S, T, G)) return 0;
    return workspace_bytes(paged_blocks(S, T, window), Hkv, D);
}

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
    // outputs cannot be written, and rows that tensor maps fetch are not described with a stride of 0: the same answer in every form
    for (const VqTensorDesc *t : {&a->q1, &a->q2, &a->out, &a->kv.k1, &a->kv.k3, &a->kv.v})
        if (expanded(*t)) return VQ_EINVAL_STRIDE;
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
    if (is_16bit(dt)) {
        int dev = 0, sms = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return VQ_EDEVICE;
        const bool few = few_form(p.max_q, G, kv.D, q8, static_cast<int64_t>(p.seqs.S) * p.Hkv, sms);
        if (!few && q8 && convert_first(p.seqs.S, T, G)) {
            p.ws_blocks = paged_blocks(p.seqs.S, T, p.W);
            const size_t need = workspace_bytes(p.ws_blocks, kv.Hkv, kv.D);
            if (p.ws_blocks * kv.Hkv <= 0x7fffffff && a->workspace != nullptr && a->workspace_bytes >= need && reinterpret_cast<uintptr_t>(a->workspace) % 256 == 0)
                p.ws = a->workspace;
        }
        return few ? launch_paged_few(p, dt, q8, s) : launch_paged_chunk(p, dt, q8, s);
    }
    return launch_paged_f32(p, q8, s);
}
