"""Forms and layouts of the paged operators that small cases pass by: the workspace on several streams and in a graph, tables longer than what
a kernel keeps of them, pools that are laid out differently, a layer's real sizes."""
import pytest
import torch

from tests.paged_cases import Case, check_attention

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def api():
    from vqtree_b200 import api as _api
    return _api


def _converts(api, c):
    """The call turns its 8-bit blocks into 16-bit floats in a workspace first."""
    return api.paged_attention_workspace_bytes(c.S, c.T, c.Hkv * c.G, c.D, c.Hkv, c.W, max(c.qs), torch.int8, c.dtype) > 0


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_calls_with_a_workspace_on_two_streams_at_once(api, dtype):
    cases = [Case(40 + i, qs, lens, 2, 4, 128, 64, 128, 128, dtype, True, True) for i, (qs, lens) in enumerate((((300, 250), (700, 400)), ((64, 500), (64, 900))))]
    assert all(_converts(api, c) for c in cases)
    alone = [c.attend(api) for c in cases]
    args = [dict(q1=c.q1.cuda(), q2=c.q2.cuda(), pages=c.pages(), block_table=c.table.cuda(), cu_q=c.cu_q.cuda(), seq_lens=c.seq_lens.cuda(), window=c.W,
                 max_q=max(c.qs), **c.far_args()) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(api.paged_attention(**args[i]))
    torch.cuda.synchronize()
    for c, want, outs in zip(cases, alone, got):
        check_attention(want, c)
        assert all(torch.equal(out, want) for out in outs)


def test_two_graphs_with_workspaces_replay_with_other_lengths(api):
    """Each graph has a workspace of its own, and its blocks go by the lengths of the replay."""
    a, b = (Case(50, qs, lens, 2, 4, 64, 64, 128, 128, F16, True, True, cols=6) for qs, lens in (((400, 200), (640, 500)), ((90, 510), (300, 640))))
    assert _converts(api, a) and _converts(api, b)
    size, snaps = max(a.pools[0].shape[0], b.pools[0].shape[0]), max(a.cnt.shape[0], b.cnt.shape[0])
    fit = lambda t, n: torch.cat((t, t.new_zeros(n - t.shape[0], *t.shape[1:]))) if t.shape[0] < n else t
    for x in (a, b):
        x.pools, x.scales = [fit(t, size) for t in x.pools], [fit(t, size) for t in x.scales]
        assert x.table.shape[1] == 10
        x.cnt, x.vsum = fit(x.cnt, snaps), fit(x.vsum, snaps)
    state = lambda x: [t.cuda() for t in (x.q1, x.q2, x.table, x.cu_q, x.seq_lens, x.cb, x.cnt, x.vsum, x.snap_table, *x.pages())]
    graphs = []
    for x in (a, b):
        s = state(x)
        run = lambda s=s: api.paged_attention(s[0], s[1], api.PagedKV(*s[9:]), *s[2:5], a.W, 600, codebook=s[5], cnt=s[6], vsum=s[7], snap_table=s[8])
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, s, out))
    for order in ((a, b), (b, a), (b, b), (a, b)):
        for (graph, s, out), x in zip(graphs, order):
            for t, new in zip(s, state(x)):
                t.copy_(new)
            out.zero_()
        for graph, _, _ in graphs:
            graph.replay()
        for (_, _, out), x in zip(graphs, order):
            check_attention(out, x)
    api.check_status()


@pytest.mark.parametrize("dtype,q8", [(F32, False), (BF16, False), (F16, False), (F32, True), (BF16, True), (F16, True)])
# single tokens and drafted ones, a chunk (8 bits: converted on the way), a long one (8 bits: through the workspace)
@pytest.mark.parametrize("qs,G", [((1, 3), 4), ((70,), 2), ((140,), 4)])
def test_windows_of_more_pages_than_a_kernel_keeps(api, dtype, q8, qs, G):
    c = Case(60, qs, [4900 + 100 * s for s in range(len(qs))], 1, G, 64, 16, 4096, 128, dtype, q8, True)
    check_attention(c.attend(api), c)
    api.check_status()


@pytest.mark.parametrize("dtype,q8", [(F32, False), (BF16, False), (F16, True)])
@pytest.mark.parametrize("qs,lens,G", [((1, 2), (400, 500), 2), ((140,), (500,), 2), ((150, 160), (500, 600), 4)])
def test_pools_that_are_laid_out_differently(api, dtype, q8, qs, lens, G):
    """Keys head by head, values token by token, raw keys in a pool of several layers; scales in yet other orders."""
    c = Case(70, qs, lens, 2, G, 64, 32, 128, 128, dtype, q8, True)
    want = c.attend(api)
    k1, v, k3, ks, vs, k3s = c.pages()
    token_major = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    layers = lambda t: torch.stack((t, t + 1, t), 1)[:, 2]
    if q8:
        ks, vs, k3s = layers(ks), vs.permute(2, 1, 0).contiguous().permute(2, 1, 0), token_major(k3s)
    pages = api.PagedKV(k1, token_major(v), layers(k3), ks, vs, k3s)
    got = c.attend(api, pages=pages)
    check_attention(got, c)
    assert torch.equal(got, want)
    new = (torch.randn(sum(qs), 2, 64, device="cuda").to(dtype) for _ in range(2))
    new = list(new)
    plain = c.pages()
    for p in (pages, plain):
        api.paged_append(*new, p, c.table.cuda(), c.cu_q.cuda(), c.seq_lens.cuda())
    for x, y in zip(pages, plain):
        assert x is None or torch.equal(x.nan_to_num(9.0) if x.is_floating_point() else x, y.nan_to_num(9.0) if y.is_floating_point() else y)
    api.check_status()


@pytest.mark.parametrize("hq,hkv,M", [(32, 32, 4), (32, 8, 2)])
def test_a_layer_of_real_size_equals_the_dense_prefill(api, hq, hkv, M):
    """6000 tokens of 32 heads of 128, window 1024, in pieces and one by one, beside the dense prefill of the whole.  Both round weights
    and outputs to bf16; the project's bar against the exact result, 2e-2, is asked of their difference."""
    from vqtree_b200 import attn_vq
    from vqtree_b200.paged_cache import PagedVectorQuantizedCache
    L, D, W, K = 6000, 128, 1024, 256
    g = torch.Generator(device="cuda").manual_seed(hkv)
    cb = torch.randn(hkv, M, K, D, generator=g, device="cuda") * D ** -0.25
    q, k, v = (torch.randn(L, h, D, generator=g, device="cuda").to(BF16) for h in (hq, hkv, hkv))
    dense = attn_vq.VectorQuantizedReRoPECache(W, cb)
    want = attn_vq.dispatch_attn_impl(*(x.transpose(0, 1)[None] for x in (q, k, v)), None, dense).reshape(L, hq, D)
    cache = PagedVectorQuantizedCache(W, cb, 120, 1, page_size=64, dtype=BF16, max_length=8192)
    s, at = cache.add_sequence(), 0
    for n in (1, 1500, 1, 7, 2048, 1, 130, 1300, 3, 1009):
        got = cache.attend([s], [n], q[at: at + n], k[at: at + n], v[at: at + n]).view(n, hq, D)
        assert (got - want[at: at + n]).abs().max().item() <= 2e-2, (at, n)
        at += n
    assert at == L
    api.check_status()


@pytest.mark.parametrize("dtype,q8", [(BF16, True), (F16, False), (F32, False)])
def test_a_call_that_fails_half_way_is_undone_to_the_bit(api, monkeypatch, dtype, q8):
    from vqtree_b200.paged_cache import PagedVectorQuantizedCache
    g = torch.Generator(device="cuda").manual_seed(9)
    cb = torch.randn(2, 2, 128, 64, generator=g, device="cuda") * 0.35
    rows = [torch.randn(1500, h, 64, generator=g, device="cuda").to(dtype) for h in (4, 2, 2)]
    part = lambda a, b: [x[a:b] for x in rows]
    made = []
    for fails in (False, True):
        cache = PagedVectorQuantizedCache(128, cb, 96, 3, page_size=32, dtype=dtype, quantized=q8, max_length=1024)
        sids = [cache.add_sequence() for _ in range(3)]
        cache.attend(sids, [400, 100, 350], *part(0, 850))
        if fails:
            held, free = [t[:3].clone() for t in (cache.cnt, cache.vsum32, cache.vsum)], cache.free_pages
            with monkeypatch.context() as m:
                m.setattr(api, "paged_attention", lambda *a, **k: (_ for _ in ()).throw(RuntimeError("out of memory")))
                with pytest.raises(RuntimeError, match="out of memory"):
                    cache.attend(sids, [300, 50, 300], *part(850, 1500))
            assert all(torch.equal(t[:3], old) for t, old in zip((cache.cnt, cache.vsum32, cache.vsum), held)) and cache.free_pages == free
        made.append(cache.attend(sids, [300, 50, 300], *part(850, 1500)))
    assert torch.equal(*made)
    api.check_status()
