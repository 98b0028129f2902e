"""The paged cache with its kernels, as a server runs them: results against the naive oracle, against the one-shot prefill, under CUDA graphs
and on other streams."""
import pytest
import torch

from tests.paged_cases import Case, check_attention
from tests.paged_scenarios import serve, whole_sequences

pytestmark = pytest.mark.gpu


# tolerances: the project's bars against the naive oracle (1e-4 fp32, 2e-2 16 bits)
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2), (torch.float16, 2e-2)])
@pytest.mark.parametrize("rerope,M,page_size", [(True, 2, 32), (False, 1, 128)])
def test_serving_equals_the_whole_prefill(dtype, tol, rerope, M, page_size):
    cb, cases, want = whole_sequences((700, 420, 129), 4, 2, 64, M, 128, 128, dtype, rerope)
    schedule = [{0: 300, 1: 5}, {1: 250, 2: 1}, {0: 1, 1: 1, 2: 1}, {0: 128, 2: 127}, {0: 3, 1: 130}, {1: 1}, {0: 200, 1: 33}] + [{0: 1}] * 68
    got, cache, _ = serve(cases, cb, schedule, 128, dtype, "cuda", rerope=rerope, page_size=page_size, num_pages=96)
    from vqtree_b200 import api
    api.check_status()
    for i in got:
        err = (got[i] - want[i][: got[i].shape[0]]).abs().max()
        assert err <= tol, (i, float(err))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_serving_with_8_bit_pages_is_the_same_however_the_tokens_come(dtype):
    """The pages hold the same values whatever chunks they were written in, so two schedules give the same result up to the rounding of
    weights and outputs (2 u |v| each); and 8-bit rows stay near the exact result."""
    cb, cases, want = whole_sequences((500, 300), 4, 2, 64, 2, 128, 128, dtype)
    a, _, _ = serve(cases, cb, [{0: 400, 1: 7}, {0: 100, 1: 293}], 128, dtype, "cuda", quantized=True, num_pages=96)
    b, _, _ = serve(cases, cb, [{0: 130}, {1: 100, 0: 1}] + [{0: 1, 1: 2}] * 100 + [{0: 269}], 128, dtype, "cuda", quantized=True, num_pages=96)
    u = torch.finfo(dtype).eps / 2
    for i in a:
        assert (a[i] - b[i]).abs().max() <= 4 * u * 5 + 1e-4           # |v| below 5
        # a value is off by half a step, 1/254 of its row's largest (below 5), a score by as much of |q| times a row of that size:
        # the mean error stays well below; codes of keys at a border may change, which moves single rows
        assert (a[i] - want[i]).abs().mean() <= 0.02


def test_cache_moves_between_dense_and_paged():
    """A prompt prefilled in one call on the dense cache, continued on pages; a paged sequence continued on the dense cache."""
    from vqtree_b200 import attn_vq
    from vqtree_b200.paged_cache import PagedVectorQuantizedCache
    dtype, W = torch.bfloat16, 128
    cb, cases, want = whole_sequences((520, 520), 4, 2, 64, 2, 128, W, dtype)
    n = 500
    stack = [torch.stack([c[j] for c in cases]).transpose(1, 2).cuda() for j in range(3)]           # [B, H, L, D]
    dense = attn_vq.VectorQuantizedReRoPECache(W, cb.cuda())
    attn_vq.dispatch_attn_impl(*(x[:, :, :n] for x in stack), None, dense)
    paged = PagedVectorQuantizedCache(W, cb, 64, 4, page_size=64, dtype=dtype, max_length=1024)
    sids = paged.adopt(dense)
    assert [paged.length(s) for s in sids] == [n, n]
    rows = lambda j, a, b: torch.cat([c[j][a:b] for c in cases]).cuda()
    got = paged.attend(sids, [10, 10], rows(0, n, 510), rows(1, n, 510), rows(2, n, 510)).view(2, 10, 4, 64)
    for i in range(2):
        assert (got[i].float().cpu() - want[i][n:510]).abs().max() <= 2e-2
    back = paged.to_dense(sids[1])
    for x in range(510, 520):
        out = attn_vq.dispatch_attn_impl(*(t[1:, :, x: x + 1] for t in stack), None, back)
        assert (out.view(4, 64).float().cpu() - want[1][x]).abs().max() <= 2e-2


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, False)])
def test_captured_calls_replay_with_other_lengths_and_tables(dtype, q8):
    """The tables and lengths are read on the device: one capture serves every step, for few tokens and for chunks."""
    from vqtree_b200 import api
    for first, second in ((((1, 1), (300, 259)), ((1, 1), (129, 640))), (((2, 1), (258, 5)), ((1, 2), (600, 130))),
                          (((140, 60), (500, 200)), ((60, 140), (640, 140)))):
        a, b = (Case(11, qs, lens, 2, 4, 64, 64, 128, 128, dtype, q8, True, cols=3) for qs, lens in (first, second))
        dev = lambda t: t.cuda()
        size = max(a.pools[0].shape[0], b.pools[0].shape[0])
        fit = lambda t, n: torch.cat((t, t.new_zeros(n - t.shape[0], *t.shape[1:]))) if t is not None and t.shape[0] < n else t
        cols, snaps = max(a.table.shape[1], b.table.shape[1]), max(x.cnt.shape[0] for x in (a, b))
        for x in (a, b):
            x.pools, x.scales = [fit(t, size) for t in x.pools], [fit(t, size) for t in x.scales]
            x.table = torch.cat((x.table, x.table.new_full((2, cols - x.table.shape[1]), -1)), 1)
            x.cnt, x.vsum = fit(x.cnt, snaps), fit(x.vsum, snaps)
        state = lambda x: [dev(t) for t in (x.q1, x.q2, x.table, x.cu_q, x.seq_lens, x.cb, x.cnt, x.vsum, x.snap_table)]
        s, pages = state(a), a.pages()
        out = torch.zeros_like(s[0])
        run = lambda: api.paged_attention(s[0], s[1], pages, s[2], s[3], s[4], a.W, max(first[0] + second[0]), codebook=s[5], cnt=s[6], vsum=s[7],
                                          snap_table=s[8], out=out)
        run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        for x in (a, b, a):
            for t, new in zip(s, state(x)):
                t.copy_(new)
            for t, new in zip(pages, x.pages()):
                if t is not None:
                    t.copy_(new)
            out.zero_()
            graph.replay()
            check_attention(out, x)
        api.check_status()


@pytest.mark.parametrize("q8", [False, True])
def test_calls_on_two_streams_at_once(q8):
    """No workspace is shared: calls of both forms on two streams give what they give alone."""
    from vqtree_b200 import api
    cases = [Case(20 + i, qs, lens, 2, 4, 128, 64, 128, 256, torch.bfloat16, q8, True) for i, (qs, lens) in
             enumerate((((1,) * 6, (300, 400, 500, 600, 700, 800)), ((130, 99), (700, 300))))]
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
    for i in (0, 1):
        for out in got[i]:
            assert torch.equal(out, alone[i])                 # the same bits: the order of additions does not depend on timing


def test_decode_graph_of_the_whole_step():
    """Append, attention in one captured graph: what a server replays per token (lengths on the device)."""
    from vqtree_b200 import api
    dtype, W = torch.bfloat16, 128
    cb, cases, want = whole_sequences((200, 170), 4, 2, 64, 1, 128, W, dtype)
    P, n0 = 64, (150, 120)
    pages = api.PagedKV.allocate(8, 2, P, 64, dtype, "cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    cat = lambda j, lo, hi: torch.cat([c[j][a:b] for c, a, b in zip(cases, lo, hi)]).cuda()
    api.paged_append(cat(1, (0, 0), n0), cat(2, (0, 0), n0), pages, table, i32(0, n0[0], sum(n0)), i32(*n0), n_pos=256)
    q, k, v = (cat(j, n0, [x + 1 for x in n0]) for j in range(3))
    cu, lens = i32(0, 1, 2), i32(*n0)

    def step():
        q1, q2 = api.paged_append(k, v, pages, table, cu, lens, q=q, const_pos=W + 1, n_pos=256)
        return api.paged_attention(q1, q2, pages, table, cu, lens, W, 1)

    graph = torch.cuda.CUDAGraph()
    before = [t.clone() for t in pages if t is not None]
    step()
    for t, old in zip((t for t in pages if t is not None), before):
        t.copy_(old)
    with torch.cuda.graph(graph):
        out = step()
    api.rope_tables(4096, 64, "cuda")                         # a longer table replaces the one the graph reads
    torch.empty(1 << 16, device="cuda").fill_(float("nan"))
    for x in range(40):
        for t, j in ((q, 0), (k, 1), (v, 2)):
            t.copy_(cat(j, [a + x for a in n0], [a + x + 1 for a in n0]))
        lens.add_(1)
        graph.replay()
        for s in range(2):
            assert (out[s].float().cpu() - want[s][n0[s] + x]).abs().max() <= 2e-2
    api.check_status()
