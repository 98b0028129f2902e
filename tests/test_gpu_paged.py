"""GPU tests of the paged cache's operators against plain implementations (tests/paged_cases.py) at the sizes and masks where they can go
wrong."""
import pytest
import torch

from tests.paged_cases import BLOCK, Case, boundary, check_attention, quantise32, rotate64
from vqtree_b200 import native

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def api():
    from vqtree_b200 import api as _api
    return _api


# ------------------------------------------------------------------------------------------- append and read

def _append_case(seed, qs, lens, Hkv, Hq, D, P, dtype, tail=3):
    g = torch.Generator().manual_seed(seed)
    T = sum(qs) + tail
    rn = lambda *s: torch.randn(*s, generator=g)
    # [T, H, D] views of one projection output: row strides other than H * D
    fused = rn(T, (Hq + 2 * Hkv) * D + 16).to(dtype)
    q, k, v = (fused[:, a * D: b * D].unflatten(1, (-1, D)) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
    MB = -(-max(lens) // P) + 1
    table = torch.randperm(len(lens) * MB, generator=g).reshape(len(lens), MB).to(torch.int32)
    pos = torch.cat([torch.arange(n - q_, n) for q_, n in zip(qs, lens)])
    seq = torch.cat([torch.full((q_,), s) for s, q_ in enumerate(qs)])
    return dict(q=q, k=k, v=v, table=table, pos=pos, seq=seq, cu_q=torch.tensor([0] + list(qs)).cumsum(0).to(torch.int32),
                lens=torch.tensor(lens, dtype=torch.int32), T=sum(qs))


def _rotate32(x, pos):
    """The documented arithmetic: fp32 tables of 64-bit angles, products and sum rounded one by one."""
    D = x.shape[-1]
    inv = 1.0 / (10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
    ang = pos.cuda().double()[:, None] * inv
    c, s = ang.cos().float().cpu()[:, None], ang.sin().float().cpu()[:, None]
    a, b = x.float().split(D // 2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("qs,lens,Hkv,Hq,D,P,rerope", [((1,), (1,), 1, 1, 64, 16, True), ((1, 1, 1, 1, 1), (1, 16, 17, 700, 128), 3, 6, 128, 16, True),
                                                       ((0, 5, 0, 130, 1, 0), (9, 5, 0, 300, 64, 33), 2, 2, 64, 32, False),
                                                       ((257, 31), (600, 31), 2, 10, 128, 128, True)])
def test_append_writes_exactly_the_new_rows(api, dtype, q8, qs, lens, Hkv, Hq, D, P, rerope):
    c = _append_case(len(qs) + P, qs, lens, Hkv, Hq, D, P, dtype)
    W = 128
    NP = int(c["table"].max()) + 1
    pages = api.PagedKV.allocate(NP, Hkv, P, D, torch.int8 if q8 else dtype, "cuda", raw_keys=rerope)
    for t in pages:
        if t is not None:
            t.fill_(7)
    before = [None if t is None else t.clone() for t in pages]
    d = lambda t: t.cuda()
    q1, q2 = api.paged_append(d(c["k"]), d(c["v"]), pages, d(c["table"]), d(c["cu_q"]), d(c["lens"]), q=d(c["q"]),
                              const_pos=W + 1 if rerope else None)
    api.check_status()
    T, pos = c["T"], c["pos"]
    want = dict(k1=_rotate32(c["k"][:T], pos), v=c["v"][:T].float(), k3=c["k"][:T].float() if rerope else None)
    page, row = c["table"][c["seq"], pos // P].long(), pos % P
    for name in ("k1", "v", "k3"):
        pool, scale = getattr(pages, name), getattr(pages, name + "_scale")
        if want[name] is None:
            assert pool is None
            continue
        rows, scales = quantise32(want[name]) if q8 else (want[name].to(dtype), None)
        exp = before[pages._fields.index(name)].cpu()
        exp[page, :, row] = rows                                    # every other row as it was
        assert torch.equal(pool.cpu(), exp), name
        if q8:
            exp = before[pages._fields.index(name + "_scale")].cpu()
            exp[page, :, row] = scales
            assert torch.equal(scale.cpu(), exp), name
    assert torch.equal(q1[:T].cpu(), _rotate32(c["q"][:T], pos).to(dtype))
    if rerope:
        assert torch.equal(q2[:T].cpu(), _rotate32(c["q"][:T], torch.full_like(pos, W + 1)).to(dtype))
    else:
        assert q2 is None


def test_append_rows_that_are_not_finite_vanish_or_are_extreme(api):
    """8-bit rows of zeros, of values whose scale would not be a normal number, at the ends of the range, with infinities and NaN."""
    D, P, n = 64, 16, 8
    k = torch.zeros(n, 1, D)
    k[1, 0] = 1e-37 * torch.linspace(-1, 1, D)                     # 1e-37 / 127 is below the normal numbers
    k[2, 0, 5], k[3, 0, 6], k[4, 0, 7] = float("inf"), float("-inf"), float("nan")
    k[5, 0] = torch.linspace(-3e38, 3e38, D)                       # not finite: the step between its ends is no fp32 number
    k[6, 0] = torch.linspace(-1e-30, 2e-30, D)
    k[7, 0] = torch.linspace(-1, 1, D) * 3.4e38
    pages = api.PagedKV.allocate(1, 1, P, D, torch.int8, "cuda", raw_keys=False)
    table, cu, lens = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    api.paged_append(k.cuda(), k.cuda(), pages, table, cu, lens, rotate=False)
    codes, scale = quantise32(k)
    for pool, sc in ((pages.k1, pages.k1_scale), (pages.v, pages.v_scale)):
        assert torch.equal(pool[0, 0, :n].cpu(), codes[:, 0])
        assert torch.equal(sc[0, 0, :n].cpu().isnan(), scale[:, 0].isnan()) and torch.equal(sc[0, 0, :n].cpu().nan_to_num(9.), scale[:, 0].nan_to_num(9.))
    back, = api.paged_read([(pages.v, pages.v_scale)], table, torch.zeros_like(lens), lens, n)
    bad = ~torch.isfinite(k[:, 0]).all(1)
    assert torch.equal(back[0, 0].cpu().isnan().any(1), bad) and bad.tolist() == [False, False, True, True, True, True, False, False]
    assert back[0, 0, :2].abs().max() == 0
    # half a step of 1/127 of the largest value, and the roundings of scale and product
    assert ((back[0, 0, 6:].cpu() - k[6:, 0]).abs() <= k[6:, 0].abs().amax(1, keepdim=True) * (0.5 / 127 + 2.0 ** -21)).all()


@pytest.mark.parametrize("dtype,q8", [(F32, False), (BF16, False), (F16, False), (F32, True), (BF16, True), (F16, True)])
@pytest.mark.parametrize("D,P,n,starts,lens", [(64, 16, 1, (0, 4, 77), (1, 4, 300)), (128, 128, 300, (-5, 0, 250), (300, 0, 400)),
                                               (128, 32, 37, (31, 63, 2), (64, 100, 2))])
def test_read_gives_rows_and_zeros(api, dtype, q8, D, P, n, starts, lens):
    g = torch.Generator().manual_seed(n)
    S, Hkv, MB = 3, 3, -(-max(lens) // P)
    table = torch.randperm(S * MB, generator=g).reshape(S, MB).to(torch.int32)
    pools = [torch.randn(S * MB, Hkv, P, D, generator=g).to(dtype) for _ in range(3)]
    scales = [None] * 3
    if q8:
        pools, scales = zip(*(quantise32(p) for p in pools))
    want = torch.zeros(3, S, Hkv, n, D)
    for i in range(3):
        val = pools[i].float() * (scales[i][..., None] if q8 else 1.0)
        for s in range(S):
            for r in range(n):
                pos = starts[s] + r
                if 0 <= pos < lens[s]:
                    want[i, s, :, r] = val[table[s, pos // P], :, pos % P]
    # pools laid out [NP, P, H, D] as well
    for lay in (lambda t: t, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        got = api.paged_read([(lay(p.cuda()), None if sc is None else lay(sc.cuda())) for p, sc in zip(pools, scales)], table.cuda(),
                             torch.tensor(starts, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), n, dtype)
        api.check_status()
        for i in range(3):
            assert torch.equal(got[i].cpu(), want[i].to(dtype))


# ------------------------------------------------------------------------------------------- attention

SHAPES = [
    # qs, lens, Hkv, G, D, P, W, MK
    pytest.param((1,), (1,), 1, 1, 64, 16, 128, 128, id="one_token_alone"),
    pytest.param((1, 1, 1, 1), (129, 130, 256, 257), 2, 4, 128, 16, 128, 128, id="decode_at_the_boundary"),
    pytest.param((1, 1, 1), (400, 1, 1023), 3, 3, 64, 32, 256, 384, id="decode_group_of_three"),
    pytest.param((1, 1), (900, 385), 2, 8, 128, 128, 128, 256, id="decode_group_of_eight"),
    pytest.param((1, 1), (500, 641), 1, 16, 128, 64, 256, 128, id="decode_group_of_sixteen"),
    pytest.param((5, 2, 1, 0), (387, 258, 300, 4), 2, 4, 64, 64, 128, 256, id="few_tokens_across_a_boundary"),
    pytest.param((4, 1), (514, 515), 2, 7, 128, 16, 256, 128, id="few_tokens_odd_group"),
    pytest.param((33, 130), (33, 391), 2, 2, 128, 32, 128, 256, id="chunk_across_two_boundaries"),
    pytest.param((257, 1, 0, 70), (600, 384, 0, 70), 1, 4, 128, 128, 128, 128, id="ragged_chunk"),
    pytest.param((200,), (513,), 2, 1, 64, 16, 256, 128, id="chunk_heads_of_64"),
    pytest.param((150, 40), (150, 640), 1, 5, 64, 64, 256, 256, id="chunk_group_of_five"),
    pytest.param((97, 3), (400, 129), 1, 40, 128, 32, 128, 128, id="chunk_wide_group"),
]


@pytest.mark.parametrize("qs,lens,Hkv,G,D,P,W,MK", SHAPES)
@pytest.mark.parametrize("dtype,q8", [(F32, False), (BF16, False), (F16, False), (F32, True), (BF16, True), (F16, True)])
@pytest.mark.parametrize("rerope", [True, False])
def test_attention(api, qs, lens, Hkv, G, D, P, W, MK, dtype, q8, rerope):
    c = Case(sum(lens) + G, qs, lens, Hkv, G, D, P, W, MK, dtype, q8, rerope, tail=2)
    out = torch.full((c.T + 2, Hkv * G, D), 5.0, dtype=dtype, device="cuda")
    c.attend(api, out=out)
    api.check_status()
    assert (out[c.T:] == 5).all()                                    # rows behind the last sequence
    check_attention(out, c)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rerope", [True, False])
@pytest.mark.parametrize("qs,lens,Hkv,G,D,P,W", [((300,), (1000,), 2, 4, 128, 64, 256), ((0, 700, 0, 600, 3), (7, 700, 0, 900, 500), 1, 8, 64, 16, 128),
                                                 ((257, 300), (257, 600), 2, 4, 128, 128, 512)])
def test_attention_8_bit_rows_converted_first_or_on_the_way(api, dtype, rerope, qs, lens, Hkv, G, D, P, W):
    """Long chunks over 8-bit pages: through the workspace and without one, the same bits."""
    c = Case(sum(lens), qs, lens, Hkv, G, D, P, W, 128, dtype, True, rerope)
    need = api.paged_attention_workspace_bytes(len(qs), c.T, Hkv * G, D, Hkv, W, max(qs), torch.int8, dtype)
    assert need > 0
    room = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")          # bytes that are no numbers, and a guard behind them
    a = c.attend(api, workspace=room[:need])
    assert (room[need:] == 255).all()
    b = c.attend(api, workspace=room[:16])                                            # too small: not used
    api.check_status()
    check_attention(a, c)
    assert torch.equal(a, b) and torch.equal(a, c.attend(api))


@pytest.mark.parametrize("dtype,q8", [(BF16, False), (F16, True), (F32, False)])
@pytest.mark.parametrize("qs,lens", [((1, 1), (300, 800)), ((3, 2), (259, 700)), ((140, 9), (600, 777))])
def test_attention_without_codebook_and_with_spare_snapshot_columns(api, dtype, q8, qs, lens):
    check_attention(Case(1, qs, lens, 2, 4, 128, 64, 128, 128, dtype, q8, True, far=False).attend(api), Case(1, qs, lens, 2, 4, 128, 64, 128, 128, dtype, q8, True, far=False))
    c = Case(2, qs, lens, 2, 4, 128, 64, 128, 128, dtype, q8, True, cols=5)
    check_attention(c.attend(api, max_q=max(qs) + 60), c)
    api.check_status()


@pytest.mark.parametrize("dtype,q8", [(BF16, False), (BF16, True), (F16, False), (F16, True), (F32, False)])
@pytest.mark.parametrize("qs,lens", [((1, 1), (300, 800)), ((150,), (700,))])
def test_attention_strided_tensors(api, dtype, q8, qs, lens):
    """Token-major pools, a pool of several layers, queries and outputs inside wider rows."""
    c = Case(3, qs, lens, 2, 2, 64, 32, 128, 256, dtype, q8, True)
    token_major = c.pages(layout=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    layered = c.pages(layout=lambda t: torch.stack((t, t, t), 1)[:, 1])
    T, Hq, D = c.q1.shape
    wide = lambda t: torch.cat((t.cuda(), t.cuda()), 2)[:, :, D:]
    for pages in (token_major, layered):
        out = torch.zeros(T, Hq, 2 * D, dtype=dtype, device="cuda")
        api.paged_attention(wide(c.q1), wide(c.q2), pages, c.table.cuda(), c.cu_q.cuda(), c.seq_lens.cuda(), c.W, max(qs), out=out[:, :, :D], **c.far_args())
        check_attention(out[:, :, :D], c)
        assert (out[:, :, D:] == 0).all()


@pytest.mark.parametrize("dtype,q8", [(BF16, False), (F16, False), (BF16, True), (F16, True), (F32, False)])
@pytest.mark.parametrize("qs,lens", [((1, 2), (400, 500)), ((140,), (500,))])
def test_attention_scores_far_apart_and_codes_without_members(api, dtype, q8, qs, lens):
    """A codeword nobody is assigned to with a towering score must not count; one real key may outweigh all others; values of very
    different sizes."""
    c = Case(4, qs, lens, 2, 2, 128, 16, 128, 256, dtype, q8, True)
    c.cnt[:, :, 3] = 0
    c.vsum[:, :, 3] = 0
    c.cb[:, 3] *= 60
    c.q1, c.q2 = (c.q1.float() * 3).to(dtype), (c.q2.float() * 3).to(dtype)
    ref, mag = c.expected()
    got = c.attend(api)[:c.T].double().cpu()
    api.check_status()
    # scores reach 3 * 16 here: three times what Case.tolerance allows for their rounding
    assert ((got - ref).abs() <= 3 * c.tolerance(ref, mag)).all()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dtype,size", [(F16, 1e-4), (F16, 100.0), (BF16, 1e-20), (BF16, 1e15)])
@pytest.mark.parametrize("qs,lens", [((1,), (300,)), ((140,), (300,))])
def test_attention_values_of_any_size(api, dtype, size, q8, qs, lens):
    """Weights of 8-bit rows carry the scale of the values: neither small nor large ones may leave the range of a half."""
    c = Case(6, qs, lens, 1, 2, 128, 32, 128, 128, dtype, q8, True, scale_v=size)
    ref, mag = c.expected()
    got = c.attend(api)[:c.T].double().cpu()
    tol = c.tolerance(ref, mag) + (2.0 ** -25 if dtype == F16 else 0.0)         # a half output's own smallest step
    assert ((got - ref).abs() <= tol).all(), float(((got - ref).abs() / tol).max())


@pytest.mark.parametrize("D,heads", [(64, 32), (128, 2)])
def test_attention_fp32_sums_over_long_windows_keep_their_bits(api, D, heads):
    """Queries of zeros weigh every key by exactly 1, so the result is the value itself.  Column d's values are 1 + 0.4 * 2^-(d % 16): added one
    by one to a sum near 2^12 each loses 0.4 of the sum's last bits, the same way every time, up to 2^-13 of the result.  Sums of 32 that are
    then added up round 32 + 4128 / 32 times, plus the division: 2^-24 each at the most."""
    n, q, W, P, S = 4128, 32, 4096, 64, 8
    col = (1 + 0.4 * 2.0 ** -(torch.arange(D) % 16).float()).cuda()
    pool = col.expand(-(-n // P), heads, P, D).contiguous()
    table = torch.arange(-(-n // P), dtype=torch.int32, device="cuda").repeat(S, 1)
    cu_q = torch.arange(0, (S + 1) * q, q, dtype=torch.int32, device="cuda")
    lens = torch.full((S,), n, dtype=torch.int32, device="cuda")
    zero = torch.zeros(S * q, heads, D, device="cuda")
    got = api.paged_attention(zero, zero, api.PagedKV(pool, pool), table, cu_q, lens, W, q)
    err = ((got - col).abs() / col).max().item()
    assert err <= (32 + n / 32 + 3) * 2.0 ** -24, err


@pytest.mark.parametrize("dtype,q8", [(F32, True), (BF16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("most", [3, 41])
def test_attention_many_sequences(api, dtype, q8, most):
    """More sequences than a warp looks up at a time, some without new tokens."""
    qs = [7 * s % most for s in range(70)]
    c = Case(13, qs, [max(1, q + 53 * s % 333) for s, q in enumerate(qs)], 1, 2, 64, 32, 128, 128, dtype, q8, True)
    check_attention(c.attend(api), c)
    api.check_status()


@pytest.mark.parametrize("dtype,q8", [(F32, False), (BF16, False), (F16, True)])
@pytest.mark.parametrize("G", [100, 128])
def test_attention_widest_groups(api, dtype, q8, G):
    c = Case(G, (3, 1), (270, 40), 1, G, 64, 64, 128, 128, dtype, q8, True)
    check_attention(c.attend(api), c)
    api.check_status()


@pytest.mark.parametrize("dtype,q8,D", [(BF16, False, 128), (F16, True, 64)])
def test_rows_behind_32_bits_of_a_pool(api, dtype, q8, D):
    """The same sequences in the first pages of a small pool and in the last of one with more than 2^32 elements: the same bits."""
    P, H, W, n, last = 128, 8, 128, 300, 2 ** 32 // (128 * 8 * D) + 4
    kind = torch.int8 if q8 else dtype
    g = torch.Generator(device="cuda").manual_seed(17)
    k, v, q = (torch.randn(n, h, D, generator=g, device="cuda", dtype=dtype) for h in (H, H, 2 * H))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    room = lambda np: [torch.empty(np, H, P, D, dtype=kind, device="cuda") for _ in range(2)]
    scale = lambda np: [torch.empty(np, H, P, device="cuda") for _ in range(2)] if q8 else [None, None]
    got = []
    for np, first in ((3, 0), (last, last - 3)):
        (k1, vp), (ks, vs) = room(np), scale(np)
        pages = api.PagedKV(k1, vp, None, ks, vs)
        table = i32(first, first + 1, first + 2)[None]
        q1, _ = api.paged_append(k, v, pages, table, i32(0, n), i32(n), q=q)
        rows = api.paged_read([(k1, ks), (vp, vs)], table, i32(0), i32(n), n, dtype)
        few = api.paged_attention(q1[-1:], q1[-1:], pages, table, i32(0, 1), i32(n), W, 1)
        chunk = api.paged_attention(q1, q1, pages, table, i32(0, n), i32(n), W, n)
        got.append(rows + [few, chunk])
        api.check_status()
    for a, b in zip(*got):
        assert torch.equal(a, b) and a.isfinite().all()


def test_attention_reports_bad_tables_and_lengths_and_stays_in_bounds(api):
    """Pages, snapshots and lengths that do not fit raise the status word; the other sequences are right."""
    for qs, lens in (((1, 1, 1), (300, 400, 500)), ((150, 140, 130), (300, 400, 500))):
        for dtype, q8 in ((BF16, False), (F16, True), (F32, False)):
            c = Case(7, qs, lens, 2, 2, 128, 64, 128, 128, dtype, q8, True)
            ref, mag = c.expected()
            keep = slice(0, qs[0])
            last = slice(qs[0] + qs[1], c.T)
            for what in ("page", "huge page", "snapshot", "length", "cu_q"):
                table, snap, cu, ln = c.table.clone(), c.snap_table.clone(), c.cu_q.clone(), c.seq_lens.clone()
                if what == "page":
                    table[1] = -1
                elif what == "huge page":
                    table[1] = 2 ** 30
                elif what == "snapshot":
                    snap[1] = 10 ** 6
                elif what == "length":
                    ln[1] = 2 ** 20
                else:
                    cu[2], cu[3] = 2 ** 30, cu[1]
                far = dict(c.far_args(), snap_table=snap.cuda())
                q1, q2 = c.q1.cuda(), c.q2.cuda()
                got = api.paged_attention(q1, q2, c.pages(), table.cuda(), cu.cuda(), ln.cuda(), c.W, max(qs), **far).double().cpu()
                with pytest.raises(native.VqError) as e:
                    api.check_status()
                assert e.value.status == -7
                tol = c.tolerance(ref, mag)
                for part in (keep,) if what == "cu_q" else (keep, last):
                    assert ((got - ref).abs() <= tol)[part].all(), what


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("qs,lens", [((1, 5), (300, 800)), ((70, 150), (300, 800)), ((700, 3), (900, 301))])
@pytest.mark.parametrize("which", [0, 2])
def test_attention_8_bit_rows_that_are_not_finite_reach_only_their_readers(api, dtype, qs, lens, which):
    """The key or value of the last sequence's last token but one was not finite: its scale is NaN.  Earlier tokens do not see it."""
    c = Case(11, qs, lens, 2, 2, 64, 32, 128, 128, dtype, True, True)
    at = lens[-1] - 2
    c.scales[which][c.table[-1, at // c.P], :, at % c.P] = float("nan")
    got = c.attend(api).double().cpu()
    ref, mag = c.expected()
    seen = min(2, qs[-1])
    clean = slice(0, c.T - seen)
    assert ((got - ref).abs() <= c.tolerance(ref, mag))[clean].all()
    assert got[c.T - seen:].isnan().all()


def test_attention_more_blocks_than_the_workspace_holds(api):
    """cu_q that decreases in between names rows more than once: the sequences' blocks may then be more than a call of that many rows can have."""
    S, q, n, W, P, G, D = 15, 1024, 1300, 128, 64, 8, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    pages = api.PagedKV(*(torch.randint(-127, 128, (21, 1, P, D), generator=g, device="cuda", dtype=torch.int8) for _ in range(3)),
                        *(torch.full((21, 1, P), 0.01, device="cuda") for _ in range(3)))
    table = torch.arange(21, dtype=torch.int32, device="cuda").repeat(S, 1)
    lens = torch.full((S,), n, dtype=torch.int32, device="cuda")
    cu_q = torch.tensor([0, q] * 8, dtype=torch.int32, device="cuda")
    q1 = torch.randn(q, G, D, generator=g, device="cuda", dtype=BF16)
    assert api.paged_attention_workspace_bytes(S, q, G, D, 1, W, q, torch.int8, BF16) > 0
    got = api.paged_attention(q1, q1, pages, table, cu_q, lens, W, q)
    with pytest.raises(native.VqError):
        api.check_status()
    assert torch.equal(got, api.paged_attention(q1, q1, pages, table[:1], cu_q[:2], lens[:1], W, q))
    api.check_status()


def test_append_reports_bad_tables_and_lengths_and_writes_nothing_for_them(api):
    D, P = 64, 16
    k = torch.randn(6, 1, D, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for table, cu, lens in ((i32(0, 9).view(2, 1), i32(0, 3, 6), i32(3, 3)), (i32(0, -1).view(2, 1), i32(0, 3, 6), i32(3, 3)),
                            (i32(0, 1).view(2, 1), i32(0, 3, 6), i32(3, 2)), (i32(0, 1).view(2, 1), i32(0, 3, 7), i32(3, 5)),
                            (i32(0, 1).view(2, 1), i32(0, 3, 6), i32(3, 40))):
        pages = api.PagedKV.allocate(2, 1, P, D, F32, "cuda", raw_keys=False)
        api.paged_append(k, k, pages, table, cu, lens)
        with pytest.raises(native.VqError):
            api.check_status()
        assert torch.equal(pages.v[0, 0, :3], k[:3, 0]) and pages.v[1].abs().max() == 0
