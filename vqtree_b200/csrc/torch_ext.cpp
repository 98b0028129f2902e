// PyTorch C++ extension over the C ABI of include/vqattn.h: registers the library's entry points as
// dispatcher operators (torch.ops.vqattn.*), so that a PyTorch program can call them like any other
// operator - under a device guard, on PyTorch's current stream, with TORCH_CHECK errors - without going
// through Python's ctypes.  Nothing here computes: every operator describes its tensors as VqTensorDesc,
// calls the C function the header declares and turns a negative status into an exception.  The operators
// write into tensors the caller passes (out-variants): the library allocates nothing, and neither does
// this file, but for the paged_*_new forms, which return new tensors.
//
// Reference interfaces behind the operators: ops/mini_vq.py:4-18 (assign_codes), ops/attn_vq.py:352-384,
// 411-417 (build_aggregates), ops/triton_fused_vq_attn.py:190-251 (prefill), README.md:8 and
// ops/attn_vq.py:128-165 (decode, cache_advance).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <optional>
#include <tuple>
#include <utility>
#include <vector>

#include "vqattn.h"

namespace {

int32_t dtype_of(const at::Tensor &t)
{
    switch (t.scalar_type()) {
        case at::kFloat: return VQ_F32;
        case at::kBFloat16: return VQ_BF16;
        case at::kHalf: return VQ_F16;
        case at::kChar: return VQ_I8;
        case at::kByte: return VQ_U8;
        case at::kUInt16: return VQ_U16;
        case at::kInt: return VQ_I32;
        case at::kLong: return VQ_I64;
        default: TORCH_CHECK(false, "vqattn: unsupported dtype ", t.scalar_type());
    }
    return -1;
}

VqTensorDesc desc(const at::Tensor &t)
{
    TORCH_CHECK(t.is_cuda(), "vqattn: CUDA tensors only (there is no CPU path)");
    TORCH_CHECK(t.dim() <= VQATTN_MAX_DIMS, "vqattn: at most ", VQATTN_MAX_DIMS, " dimensions");
    VqTensorDesc d{};
    d.ptr = t.data_ptr();
    d.dtype = dtype_of(t);
    d.ndim = static_cast<int32_t>(t.dim());
    for (int64_t i = 0; i < t.dim(); ++i) {
        d.shape[i] = t.size(i);
        d.stride[i] = t.stride(i);
    }
    d.device = static_cast<int32_t>(t.get_device());
    return d;
}

VqTensorDesc desc(const std::optional<at::Tensor> &t)
{
    if (t.has_value() && t->defined()) return desc(*t);
    VqTensorDesc d{};
    d.device = -1;
    return d;
}

void check(int status, const char *where)
{
    TORCH_CHECK(status == VQ_OK, where, ": ", vqattn_status_string(status), " (status ", status, ")");
}

void *stream_of(const at::Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

int32_t *word_of(const std::optional<at::Tensor> &w)
{
    if (!w.has_value() || !w->defined()) return nullptr;
    TORCH_CHECK(w->is_cuda() && w->scalar_type() == at::kInt && w->numel() >= 1, "vqattn: status word must be a CUDA int32 tensor");
    return w->data_ptr<int32_t>();
}

struct Workspace {
    void *ptr = nullptr;
    size_t bytes = 0;
    explicit Workspace(const std::optional<at::Tensor> &w)
    {
        if (w.has_value() && w->defined()) {
            TORCH_CHECK(w->is_cuda() && w->is_contiguous(), "vqattn: workspace must be a contiguous CUDA tensor");
            ptr = w->data_ptr();
            bytes = static_cast<size_t>(w->numel()) * w->element_size();
        }
    }
};

// codes[B,Hkv,L,M] <- assignment of k[B,Hkv,L,D] against codebooks[Hkv,M,K,D]; with a workspace of
// assign_workspace_bytes(...) the scores run on the tensor cores (same codes)
void assign_codes(const at::Tensor &k, const at::Tensor &codebooks, const std::optional<at::Tensor> &bias, at::Tensor codes,
                  const std::optional<at::Tensor> &workspace, const std::optional<at::Tensor> &status_word)
{
    const c10::cuda::CUDAGuard guard(k.device());
    VqTensorDesc dk = desc(k), dc = desc(codebooks), db = desc(bias), dout = desc(codes);
    const Workspace ws(workspace);
    const VqTensorDesc *pb = (bias.has_value() && bias->defined()) ? &db : nullptr;
    if (ws.ptr != nullptr)
        check(vqattn_assign_codes_ws(&dk, &dc, pb, &dout, ws.ptr, ws.bytes, word_of(status_word), stream_of(k)), "vqattn::assign_codes");
    else
        check(vqattn_assign_codes(&dk, &dc, pb, &dout, stream_of(k)), "vqattn::assign_codes");
}

int64_t assign_workspace_bytes(int64_t B, int64_t Hkv, int64_t L, int64_t M, int64_t K, int64_t D)
{
    return static_cast<int64_t>(vqattn_assign_workspace_bytes(B, Hkv, L, M, K, D));
}

// cnt[B,Hkv,NB,MK], vsum[B,Hkv,NB,MK,D] <- per-block aggregates; state_cnt / state_vsum (both or neither): the fp32
// aggregates of the first state_blocks * 128 keys from the same pass
void build_aggregates(const at::Tensor &codes, const at::Tensor &v, int64_t K, at::Tensor cnt, at::Tensor vsum,
                      const std::optional<at::Tensor> &state_cnt, const std::optional<at::Tensor> &state_vsum, int64_t state_blocks,
                      const std::optional<at::Tensor> &workspace, const std::optional<at::Tensor> &status_word)
{
    const c10::cuda::CUDAGuard guard(v.device());
    VqTensorDesc dc = desc(codes), dv = desc(v), dcnt = desc(cnt), dvs = desc(vsum);
    const Workspace ws(workspace);
    const bool with_state = state_cnt.has_value() && state_cnt->defined();
    TORCH_CHECK(with_state == (state_vsum.has_value() && state_vsum->defined()), "vqattn::build_aggregates: pass both state tensors or neither");
    if (with_state) {
        VqTensorDesc dsc = desc(state_cnt), dsv = desc(state_vsum);
        check(vqattn_build_aggregates_state(&dc, &dv, static_cast<int32_t>(K), &dcnt, &dvs, &dsc, &dsv, state_blocks, ws.ptr, ws.bytes,
                                            word_of(status_word), stream_of(v)),
              "vqattn::build_aggregates");
    } else {
        check(vqattn_build_aggregates_ws(&dc, &dv, static_cast<int32_t>(K), &dcnt, &dvs, ws.ptr, ws.bytes, word_of(status_word), stream_of(v)),
              "vqattn::build_aggregates");
    }
}

int64_t aggregates_workspace_bytes(int64_t B, int64_t Hkv, int64_t NB, int64_t M, int64_t K)
{
    return static_cast<int64_t>(vqattn_aggregates_workspace_bytes(B, Hkv, NB, M, K));
}

// out[B,Hq,L,D] <- fused prefill attention (window keys exactly, older keys through the aggregates)
void prefill(const at::Tensor &q1, const at::Tensor &q2, const at::Tensor &k1, const at::Tensor &k3, const at::Tensor &v,
             const std::optional<at::Tensor> &codebook, const std::optional<at::Tensor> &cnt, const std::optional<at::Tensor> &vsum,
             int64_t window, double scale, int64_t impl, at::Tensor out, const std::optional<at::Tensor> &lse2,
             const std::optional<at::Tensor> &status_word)
{
    const c10::cuda::CUDAGuard guard(q1.device());
    VqPrefillArgs a{};
    a.q1 = desc(q1); a.q2 = desc(q2); a.k1 = desc(k1); a.k3 = desc(k3); a.v = desc(v);
    a.codebook = desc(codebook); a.cnt = desc(cnt); a.vsum = desc(vsum);
    a.out = desc(out);
    a.lse2 = desc(lse2);
    a.window = window;
    a.scale = static_cast<float>(scale);
    a.impl = static_cast<int32_t>(impl);
    a.status_word = word_of(status_word);
    check(vqattn_prefill(&a, stream_of(q1)), "vqattn::prefill");
}

// out[B,Hq,D] <- one decode step over the window caches and the aggregates
void decode(const at::Tensor &q1, const at::Tensor &q2, const at::Tensor &k1_win, const at::Tensor &k3_win, const at::Tensor &v_win,
            const std::optional<at::Tensor> &codebook, const std::optional<at::Tensor> &cnt, const std::optional<at::Tensor> &vsum,
            int64_t n_valid, int64_t n_bd, double scale, at::Tensor workspace, at::Tensor out, const std::optional<at::Tensor> &status_word)
{
    const c10::cuda::CUDAGuard guard(q1.device());
    VqDecodeArgs a{};
    a.q1 = desc(q1); a.q2 = desc(q2); a.k1_win = desc(k1_win); a.k3_win = desc(k3_win); a.v_win = desc(v_win);
    a.codebook = desc(codebook); a.cnt = desc(cnt); a.vsum = desc(vsum);
    a.out = desc(out);
    a.n_valid = n_valid;
    a.n_bd = n_bd;
    a.use_far = (codebook.has_value() && codebook->defined()) ? 1 : 0;
    a.scale = static_cast<float>(scale);
    const std::optional<at::Tensor> ws_t{workspace};
    const Workspace ws(ws_t);
    a.workspace = ws.ptr;
    a.workspace_bytes = ws.bytes;
    a.status_word = word_of(status_word);
    check(vqattn_decode(&a, stream_of(q1)), "vqattn::decode");
}

int64_t decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D)
{
    return static_cast<int64_t>(vqattn_decode_workspace_bytes(B, Hq, Hkv, D));
}

// cnt[B,Hkv,MK], vsum_f32[B,Hkv,MK,D] (+ 16-bit copy) += the keys codes[B,Hkv,n,M] / v_new[B,Hkv,n,D] that left the window
void cache_advance(const at::Tensor &codes, const at::Tensor &v_new, int64_t K, at::Tensor cnt, at::Tensor vsum_f32,
                   const std::optional<at::Tensor> &vsum_act, const std::optional<at::Tensor> &status_word)
{
    const c10::cuda::CUDAGuard guard(v_new.device());
    VqTensorDesc dc = desc(codes), dv = desc(v_new), dcnt = desc(cnt), dvs = desc(vsum_f32), dva = desc(vsum_act);
    VqTensorDesc *pva = (vsum_act.has_value() && vsum_act->defined()) ? &dva : nullptr;
    check(vqattn_cache_advance(&dc, &dv, static_cast<int32_t>(K), &dcnt, &dvs, pva, word_of(status_word), stream_of(v_new)),
          "vqattn::cache_advance");
}

// ---- the paged cache.  The plain forms write into their arguments and raise; the *_status forms return the C status instead (what
// vqtree_b200/api.py turns into its own exception), and the *_new forms allocate the outputs too (three times as fast here as from Python).

VqTensorDesc any_desc(const at::Tensor &t)         // host tensors too: the C function answers VQ_EDEVICE for them
{
    if (t.is_cuda()) return desc(t);
    VqTensorDesc d{};
    TORCH_CHECK(t.dim() <= VQATTN_MAX_DIMS, "vqattn: at most ", VQATTN_MAX_DIMS, " dimensions");
    d.ptr = t.numel() > 0 ? t.data_ptr() : reinterpret_cast<void *>(16);
    d.dtype = dtype_of(t);
    d.ndim = static_cast<int32_t>(t.dim());
    for (int64_t i = 0; i < t.dim(); ++i) {
        d.shape[i] = t.size(i);
        d.stride[i] = t.stride(i);
    }
    d.device = -1;
    return d;
}
VqTensorDesc any_desc(const std::optional<at::Tensor> &t)
{
    return t.has_value() && t->defined() ? any_desc(*t) : desc(t);
}

using OptTensor = std::optional<at::Tensor>;

// a CUDA tensor of another device than the call's: what goes to the C function as a bare pointer, which it cannot check
bool elsewhere(const OptTensor &t, const at::Tensor &call) { return t.has_value() && t->defined() && t->is_cuda() && t->get_device() != call.get_device(); }

VqPagedKv paged_kv(const at::Tensor &k1, const at::Tensor &v, const OptTensor &k3, const OptTensor &k1_scale, const OptTensor &v_scale,
                   const OptTensor &k3_scale, const at::Tensor &table, const at::Tensor &cu_q, const at::Tensor &lens)
{
    VqPagedKv kv{};
    kv.k1 = any_desc(k1); kv.v = any_desc(v); kv.k3 = any_desc(k3);
    kv.k1_scale = any_desc(k1_scale); kv.v_scale = any_desc(v_scale); kv.k3_scale = any_desc(k3_scale);
    kv.table = any_desc(table); kv.cu_q = any_desc(cu_q); kv.lens = any_desc(lens);
    return kv;
}

// pages <- new tokens k, v [T,Hkv,D] (rotated when there are tables), q1 / q2 <- q [T,Hq,D] rotated
int64_t paged_append_status(const at::Tensor &k, const at::Tensor &v, at::Tensor k1, at::Tensor v_pages, const OptTensor &k3,
                            const OptTensor &k1_scale, const OptTensor &v_scale, const OptTensor &k3_scale, const at::Tensor &table,
                            const at::Tensor &cu_q, const at::Tensor &lens, const OptTensor &q, const OptTensor &q1, const OptTensor &q2,
                            const OptTensor &cos_tab, const OptTensor &sin_tab, int64_t const_pos, const OptTensor &status_word)
{
    if (!k.is_cuda() || elsewhere(cos_tab, k) || elsewhere(sin_tab, k) || elsewhere(status_word, k)) return VQ_EDEVICE;
    const c10::cuda::CUDAGuard guard(k.device());
    VqPagedAppendArgs a{};
    a.kv = paged_kv(k1, v_pages, k3, k1_scale, v_scale, k3_scale, table, cu_q, lens);
    a.k = any_desc(k); a.v = any_desc(v); a.q = any_desc(q); a.q1 = any_desc(q1); a.q2 = any_desc(q2);
    if (cos_tab.has_value() && cos_tab->defined()) {
        TORCH_CHECK(sin_tab.has_value() && cos_tab->is_cuda() && sin_tab->is_cuda() && cos_tab->scalar_type() == at::kFloat &&
                        sin_tab->scalar_type() == at::kFloat && cos_tab->is_contiguous() && sin_tab->is_contiguous() &&
                        cos_tab->sizes() == sin_tab->sizes() && cos_tab->dim() == 2 && 2 * cos_tab->size(1) == k.size(-1),
                    "vqattn: cos / sin tables are contiguous CUDA float32 [n_pos, D / 2]");
        a.cos_tab = cos_tab->data_ptr<float>();
        a.sin_tab = sin_tab->data_ptr<float>();
        a.n_pos = cos_tab->size(0);
    }
    a.const_pos = const_pos;
    a.status_word = word_of(status_word);
    return vqattn_paged_append(&a, stream_of(k));
}

// out [S,Hkv,n,D] <- rows [start, start + n) of every sequence in a pool; up to three pools
int64_t paged_read_status(const at::Tensor &pool0, const OptTensor &scale0, at::Tensor out0, const OptTensor &pool1, const OptTensor &scale1,
                          const OptTensor &out1, const OptTensor &pool2, const OptTensor &scale2, const OptTensor &out2, const at::Tensor &table,
                          const at::Tensor &start, const at::Tensor &lens, const OptTensor &status_word)
{
    if (!pool0.is_cuda() || elsewhere(status_word, pool0)) return VQ_EDEVICE;
    const c10::cuda::CUDAGuard guard(pool0.device());
    VqPagedReadArgs a{};
    a.pool[0] = any_desc(pool0); a.pool[1] = any_desc(pool1); a.pool[2] = any_desc(pool2);
    a.scale[0] = any_desc(scale0); a.scale[1] = any_desc(scale1); a.scale[2] = any_desc(scale2);
    a.out[0] = any_desc(out0); a.out[1] = any_desc(out1); a.out[2] = any_desc(out2);
    a.table = any_desc(table); a.start = any_desc(start); a.lens = any_desc(lens);
    a.status_word = word_of(status_word);
    return vqattn_paged_read(&a, stream_of(pool0));
}

// out [T,Hq,D] <- attention of the new tokens over their pages and, before the boundary, over the snapshots
int64_t paged_attention_status(const at::Tensor &q1, const at::Tensor &q2, const at::Tensor &k1, const at::Tensor &v_pages, const OptTensor &k3,
                               const OptTensor &k1_scale, const OptTensor &v_scale, const OptTensor &k3_scale, const at::Tensor &table,
                               const at::Tensor &cu_q, const at::Tensor &lens, const OptTensor &codebook, const OptTensor &cnt,
                               const OptTensor &vsum, const OptTensor &snap_table, int64_t window, int64_t max_q, double scale, at::Tensor out,
                               const OptTensor &workspace, const OptTensor &status_word)
{
    if (!q1.is_cuda() || elsewhere(workspace, q1) || elsewhere(status_word, q1)) return VQ_EDEVICE;
    const c10::cuda::CUDAGuard guard(q1.device());
    VqPagedAttentionArgs a{};
    a.kv = paged_kv(k1, v_pages, k3, k1_scale, v_scale, k3_scale, table, cu_q, lens);
    a.q1 = any_desc(q1); a.q2 = any_desc(q2); a.out = any_desc(out);
    a.codebook = any_desc(codebook); a.cnt = any_desc(cnt); a.vsum = any_desc(vsum); a.snap_table = any_desc(snap_table);
    a.window = window;
    a.max_q = max_q;
    a.scale = static_cast<float>(scale);
    a.status_word = word_of(status_word);
    const Workspace ws(workspace);
    a.workspace = ws.ptr;
    a.workspace_bytes = ws.bytes;
    return vqattn_paged_attention(&a, stream_of(q1));
}

// a workspace for the call, undefined where it would use none
OptTensor paged_workspace(const at::Tensor &q1, const at::Tensor &k1, const at::Tensor &table, int64_t window, int64_t max_q)
{
    if (k1.scalar_type() != at::kChar || q1.dim() != 3 || k1.dim() != 4 || table.dim() != 2 || !q1.is_cuda()) return {};
    const size_t n = vqattn_paged_attention_workspace_bytes(table.size(0), q1.size(0), q1.size(1), k1.size(1), q1.size(2), window, max_q, VQ_I8,
                                                            dtype_of(q1));
    return n ? OptTensor(at::empty({static_cast<int64_t>(n)}, q1.options().dtype(at::kByte))) : OptTensor();
}

std::tuple<at::Tensor, at::Tensor, int64_t> paged_append_new(const at::Tensor &k, const at::Tensor &v, at::Tensor k1, at::Tensor v_pages,
                                                             const OptTensor &k3, const OptTensor &k1_scale, const OptTensor &v_scale,
                                                             const OptTensor &k3_scale, const at::Tensor &table, const at::Tensor &cu_q,
                                                             const at::Tensor &lens, const at::Tensor &q, bool two, const OptTensor &cos_tab,
                                                             const OptTensor &sin_tab, int64_t const_pos, const OptTensor &status_word)
{
    const at::Tensor q1 = at::empty(q.sizes(), q.options()), q2 = two ? at::empty(q.sizes(), q.options()) : q1;
    const int64_t status = paged_append_status(k, v, std::move(k1), std::move(v_pages), k3, k1_scale, v_scale, k3_scale, table, cu_q, lens, q, q1,
                                               two ? OptTensor(q2) : OptTensor(), cos_tab, sin_tab, const_pos, status_word);
    return {q1, two ? q2 : at::Tensor(at::empty({0}, q.options())), status};
}

std::tuple<std::vector<at::Tensor>, int64_t> paged_read_new(at::TensorList pools, const c10::List<OptTensor> &scales, const at::Tensor &table,
                                                            const at::Tensor &start, const at::Tensor &lens, int64_t n, at::ScalarType dtype,
                                                            const OptTensor &status_word)
{
    TORCH_CHECK(!pools.empty() && pools.size() <= 3 && pools.size() == scales.size(), "vqattn: one to three pools, a scale or none for each");
    TORCH_CHECK(pools[0].dim() == 4 && table.dim() == 2, "vqattn: pools [NP,Hkv,P,D], table [S,MB]");
    std::vector<at::Tensor> outs;
    OptTensor pool[3], scale[3], out[3];
    for (size_t i = 0; i < pools.size(); ++i) {
        outs.push_back(at::empty({table.size(0), pools[0].size(1), n, pools[0].size(3)}, pools[0].options().dtype(dtype)));
        pool[i] = pools[i];
        scale[i] = scales.get(i);
        out[i] = outs.back();
    }
    const int64_t status = paged_read_status(pools[0], scale[0], outs[0], pool[1], scale[1], out[1], pool[2], scale[2], out[2], table, start, lens,
                                             status_word);
    return {outs, status};
}

std::tuple<at::Tensor, int64_t> paged_attention_new(const at::Tensor &q1, const at::Tensor &q2, const at::Tensor &k1, const at::Tensor &v_pages,
                                                    const OptTensor &k3, const OptTensor &k1_scale, const OptTensor &v_scale,
                                                    const OptTensor &k3_scale, const at::Tensor &table, const at::Tensor &cu_q,
                                                    const at::Tensor &lens, const OptTensor &codebook, const OptTensor &cnt, const OptTensor &vsum,
                                                    const OptTensor &snap_table, int64_t window, int64_t max_q, double scale,
                                                    const OptTensor &status_word)
{
    const at::Tensor out = at::empty(q1.sizes(), q1.options());
    return {out, paged_attention_status(q1, q2, k1, v_pages, k3, k1_scale, v_scale, k3_scale, table, cu_q, lens, codebook, cnt, vsum, snap_table, window,
                                        max_q, scale, out, paged_workspace(q1, k1, table, window, max_q), status_word)};
}

// the raising forms
template <auto F> struct Raising;
template <typename... A, int64_t (*F)(A...)> struct Raising<F> {
    static void call(A... args) { check(static_cast<int>(F(std::forward<A>(args)...)), "vqattn::paged"); }
};

int64_t paged_attention_workspace_bytes(int64_t S, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t window, int64_t max_q,
                                        at::ScalarType pool, at::ScalarType act)
{
    auto code = [](at::ScalarType t) { return t == at::kChar ? VQ_I8 : t == at::kBFloat16 ? VQ_BF16 : t == at::kHalf ? VQ_F16 : VQ_F32; };
    return static_cast<int64_t>(vqattn_paged_attention_workspace_bytes(S, T, Hq, Hkv, D, window, max_q, code(pool), code(act)));
}

int64_t abi_version() { return vqattn_version(); }

}  // namespace

TORCH_LIBRARY(vqattn, m)
{
    m.def("abi_version() -> int", &abi_version);
    m.def("assign_workspace_bytes(int B, int Hkv, int L, int M, int K, int D) -> int", &assign_workspace_bytes);
    m.def("aggregates_workspace_bytes(int B, int Hkv, int NB, int M, int K) -> int", &aggregates_workspace_bytes);
    m.def("decode_workspace_bytes(int B, int Hq, int Hkv, int D) -> int", &decode_workspace_bytes);
    m.def("paged_attention_workspace_bytes(int S, int T, int Hq, int Hkv, int D, int window, int max_q, ScalarType pool, ScalarType act) -> int",
          &paged_attention_workspace_bytes);
    m.def("assign_codes(Tensor k, Tensor codebooks, Tensor? bias, Tensor(a!) codes, Tensor(b!)? workspace, Tensor(c!)? status_word) -> ()");
    m.def("build_aggregates(Tensor codes, Tensor v, int K, Tensor(a!) cnt, Tensor(b!) vsum, Tensor(c!)? state_cnt, Tensor(d!)? state_vsum, "
          "int state_blocks, Tensor(e!)? workspace, Tensor(f!)? status_word) -> ()");
    m.def("prefill(Tensor q1, Tensor q2, Tensor k1, Tensor k3, Tensor v, Tensor? codebook, Tensor? cnt, Tensor? vsum, int window, "
          "float scale, int impl, Tensor(a!) out, Tensor(b!)? lse2, Tensor(c!)? status_word) -> ()");
    m.def("decode(Tensor q1, Tensor q2, Tensor k1_win, Tensor k3_win, Tensor v_win, Tensor? codebook, Tensor? cnt, Tensor? vsum, "
          "int n_valid, int n_bd, float scale, Tensor(a!) workspace, Tensor(b!) out, Tensor(c!)? status_word) -> ()");
    m.def("cache_advance(Tensor codes, Tensor v_new, int K, Tensor(a!) cnt, Tensor(b!) vsum_f32, Tensor(c!)? vsum_act, "
          "Tensor(d!)? status_word) -> ()");
    m.def("paged_append(Tensor k, Tensor v, Tensor(a!) k1, Tensor(b!) v_pages, Tensor(c!)? k3, Tensor(d!)? k1_scale, Tensor(e!)? v_scale, "
          "Tensor(f!)? k3_scale, Tensor table, Tensor cu_q, Tensor lens, Tensor? q, Tensor(g!)? q1, Tensor(h!)? q2, Tensor? cos_tab, "
          "Tensor? sin_tab, int const_pos, Tensor(i!)? status_word) -> ()");
    m.def("paged_append_status(Tensor k, Tensor v, Tensor(a!) k1, Tensor(b!) v_pages, Tensor(c!)? k3, Tensor(d!)? k1_scale, Tensor(e!)? v_scale, "
          "Tensor(f!)? k3_scale, Tensor table, Tensor cu_q, Tensor lens, Tensor? q, Tensor(g!)? q1, Tensor(h!)? q2, Tensor? cos_tab, "
          "Tensor? sin_tab, int const_pos, Tensor(i!)? status_word) -> int");
    m.def("paged_read(Tensor pool0, Tensor? scale0, Tensor(a!) out0, Tensor? pool1, Tensor? scale1, Tensor(b!)? out1, Tensor? pool2, Tensor? scale2, "
          "Tensor(c!)? out2, Tensor table, Tensor start, Tensor lens, Tensor(d!)? status_word) -> ()");
    m.def("paged_read_status(Tensor pool0, Tensor? scale0, Tensor(a!) out0, Tensor? pool1, Tensor? scale1, Tensor(b!)? out1, Tensor? pool2, Tensor? scale2, "
          "Tensor(c!)? out2, Tensor table, Tensor start, Tensor lens, Tensor(d!)? status_word) -> int");
    m.def("paged_attention(Tensor q1, Tensor q2, Tensor k1, Tensor v_pages, Tensor? k3, Tensor? k1_scale, Tensor? v_scale, Tensor? k3_scale, Tensor table, "
          "Tensor cu_q, Tensor lens, Tensor? codebook, Tensor? cnt, Tensor? vsum, Tensor? snap_table, int window, int max_q, float scale, "
          "Tensor(a!) out, Tensor(b!)? workspace, Tensor(c!)? status_word) -> ()");
    m.def("paged_attention_status(Tensor q1, Tensor q2, Tensor k1, Tensor v_pages, Tensor? k3, Tensor? k1_scale, Tensor? v_scale, Tensor? k3_scale, Tensor table, "
          "Tensor cu_q, Tensor lens, Tensor? codebook, Tensor? cnt, Tensor? vsum, Tensor? snap_table, int window, int max_q, float scale, "
          "Tensor(a!) out, Tensor(b!)? workspace, Tensor(c!)? status_word) -> int");
    m.def("paged_append_new(Tensor k, Tensor v, Tensor(a!) k1, Tensor(b!) v_pages, Tensor(c!)? k3, Tensor(d!)? k1_scale, Tensor(e!)? v_scale, "
          "Tensor(f!)? k3_scale, Tensor table, Tensor cu_q, Tensor lens, Tensor q, bool two, Tensor? cos_tab, Tensor? sin_tab, int const_pos, "
          "Tensor(g!)? status_word) -> (Tensor, Tensor, int)");
    m.def("paged_read_new(Tensor[] pools, Tensor?[] scales, Tensor table, Tensor start, Tensor lens, int n, ScalarType dtype, "
          "Tensor(a!)? status_word) -> (Tensor[], int)");
    m.def("paged_attention_new(Tensor q1, Tensor q2, Tensor k1, Tensor v_pages, Tensor? k3, Tensor? k1_scale, Tensor? v_scale, Tensor? k3_scale, "
          "Tensor table, Tensor cu_q, Tensor lens, Tensor? codebook, Tensor? cnt, Tensor? vsum, Tensor? snap_table, int window, int max_q, "
          "float scale, Tensor(a!)? status_word) -> (Tensor, int)");
}

TORCH_LIBRARY_IMPL(vqattn, CUDA, m)
{
    m.impl("assign_codes", &assign_codes);
    m.impl("build_aggregates", &build_aggregates);
    m.impl("prefill", &prefill);
    m.impl("decode", &decode);
    m.impl("cache_advance", &cache_advance);
    m.impl("paged_append_new", &paged_append_new);
    m.impl("paged_read_new", &paged_read_new);
    m.impl("paged_attention_new", &paged_attention_new);
    m.impl("paged_append", &Raising<&paged_append_status>::call);
    m.impl("paged_append_status", &paged_append_status);
    m.impl("paged_read", &Raising<&paged_read_status>::call);
    m.impl("paged_read_status", &paged_read_status);
    m.impl("paged_attention", &Raising<&paged_attention_status>::call);
    m.impl("paged_attention_status", &paged_attention_status);
}
