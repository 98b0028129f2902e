"""The operators of the paged cache as cases that can be timed: appending tokens to pages, reading pages back, and the attention of new
tokens over them.

Kinds of pass (``case["kind"]``):

``append``  new tokens of S sequences into the pages of a cache: keys rotated to their positions, raw keys, values, queries rotated on
            the way.  8-bit pages are read back in the same pass, so that what they stand for is an output.
``read``    rows of S sequences out of their pages, dense (a block that leaves the window; a sequence that leaves the cache)
``attend``  attention of the new tokens over window pages and per-code sums of everything older

Definitions.  A sequence has n tokens, the last q of them new.  The query at position i attends, with window W and
b = max(0, (i - W) // 128 * 128), to keys [max(0, i - W), i] by q1.k1, to keys [b, max(0, i - W)) by q2.k3, and to everything before b
through counts and value sums per code: score q2.C[r], weight vsum[r] in the numerator and cnt[r] in the denominator; codes without
members do not count.  Without ReRoPE q2 is q1 and k3 is k1.  Token j of a sequence lies in page ``table[s, j // P]`` at row j % P; the
sums of boundary b in snapshot ``snaps[s, b // 128 % snaps.shape[1]]``.
8-bit rows: scale = max|x| * (1/127), code = round-to-even(x * (1 / scale)), all in 32 bits; the value is code * scale.

q, k, v ~ N(0, 1), codebook entries ~ N(0, D^-1/2); counts and sums are those of as many members as the context has older tokens.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
BASE = 10000.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # ---- appending
        # a step of a server: one token of each of 48 conversations, grouped-query heads, 8-bit pages
        dict(name="append_step_q8", kind="append", dtype="bf16", q8=True, S=48, q=1, ctx=9000, ragged=True, Hq=32, Hkv=8, D=128, P=64, W=1024, rerope=True),
        # a prompt's piece of 2048 tokens, one sequence, 7B heads, pages in the activations' type
        dict(name="append_chunk_bf16", kind="append", dtype="bf16", q8=False, S=1, q=2048, ctx=6144, ragged=False, Hq=32, Hkv=32, D=128, P=128, W=1024, rerope=True),
        # second turns of twelve conversations, odd lengths, 8 bits, plain rotary positions
        dict(name="append_turns_q8", kind="append", dtype="fp16", q8=True, S=12, q=1999, ctx=12001, ragged=True, Hq=32, Hkv=8, D=128, P=16, W=2048, rerope=False),
        # ---- reading back
        # the blocks of three sequences that leave the window in one step: raw keys and values, to be quantised into codes
        dict(name="read_blocks_q8", kind="read", dtype="bf16", q8=True, S=3, n=128, ctx=9000, ragged=True, Hkv=8, D=128, P=64),
        # sixteen sequences leave the cache with their windows
        dict(name="read_windows_q8", kind="read", dtype="fp16", q8=True, S=16, n=2303, ctx=20000, ragged=True, Hkv=32, D=128, P=32),
        # ---- attention, single tokens
        # one conversation, one token
        dict(name="decode_b1", kind="attend", dtype="bf16", q8=False, S=1, q=1, ctx=4171, ragged=False, Hq=32, Hkv=8, D=128, P=128, W=1024, M=4, K=256, rerope=True),
        # sixteen sequences near context 32768, 7B heads, 8-bit window
        dict(name="decode_b16_q8", kind="attend", dtype="bf16", q8=True, S=16, q=1, ctx=32768, ragged=True, Hq=32, Hkv=32, D=128, P=128, W=1024, M=4, K=256, rerope=True),
        # a full server: 64 sequences, grouped-query heads, long window, eight codebooks
        dict(name="decode_b64_gqa", kind="attend", dtype="bf16", q8=False, S=64, q=1, ctx=60000, ragged=True, Hq=32, Hkv=8, D=128, P=64, W=2048, M=8, K=256, rerope=True),
        # ---- attention, chunks
        # five drafted tokens of each of eight sequences, half precision, heads of 64
        dict(name="draft_5_fp16", kind="attend", dtype="fp16", q8=False, S=8, q=5, ctx=3001, ragged=False, Hq=16, Hkv=4, D=64, P=16, W=512, M=2, K=256, rerope=False),
        # full precision: a chunk of odd length over a short window
        dict(name="chunk_fp32", kind="attend", dtype="fp32", q8=False, S=2, q=201, ctx=1100, ragged=True, Hq=8, Hkv=8, D=64, P=32, W=128, M=2, K=256, rerope=True),
        # second turns of six conversations, 8-bit window
        dict(name="chunk_turns_q8", kind="attend", dtype="bf16", q8=True, S=6, q=700, ctx=9001, ragged=True, Hq=32, Hkv=8, D=128, P=64, W=1024, M=4, K=256, rerope=True),
        # a piece of a long prompt: 4096 tokens at context 32768, 7B heads
        dict(name="chunk_4k", kind="attend", dtype="bf16", q8=False, S=1, q=4096, ctx=32768, ragged=False, Hq=32, Hkv=32, D=128, P=128, W=1024, M=4, K=256, rerope=True),
    ]


# ------------------------------------------------------------------------------------------- more of the same ranges

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["append", "read", "attend", "attend", "attend", "attend"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
        c = dict(kind=kind, dtype=dtype, q8=rng.random() < 0.5, S=_log_int(rng, 1, 64), ragged=rng.random() < 0.7, Hkv=rng.choice([1, 2, 4, 8, 8, 16, 32]),
                 D=rng.choice([64, 128, 128]), P=rng.choice([16, 32, 64, 128]), ctx=_log_int(rng, 40, 60000))
        if kind == "read":
            c["n"] = _log_int(rng, 1, 2400)
        else:
            c["q"] = min(c["ctx"], rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 3000), _log_int(rng, 17, 3000)]))
            c["Hq"] = c["Hkv"] * rng.choice([1, 2, 3, 4, 4, 5, 8])
            c["W"] = BLOCK * rng.choice([1, 2, 4, 8, 8, 16])
            c["rerope"] = rng.random() < 0.6
        if kind == "attend":
            c["M"], c["K"] = rng.choice([(1, 128), (1, 1024), (2, 128), (2, 256), (4, 256), (4, 256), (8, 256), (4, 512)])
        if c.get("Hq", 1) > 64:
            continue
        w = work(c)
        # full precision runs on the regular cores: its drawn sizes stay small
        if w["flops"] < (1.0e10 if dtype == "fp32" else 1.3e11) and w["bytes"] < 6.0e8:
            return c


# ------------------------------------------------------------------------------------------- lengths

def _lengths(c):
    """(new tokens, length with them) of every sequence: from the case alone."""
    qs, ns = [], []
    for s in range(c["S"]):
        f = (0.31 + s * 0.6180339887) % 1.0 if c["ragged"] else 0.0
        q = max(1, round(c.get("q", 1) * (1.0 - 0.9 * f)))
        qs.append(q)
        ns.append(max(q, round(c["ctx"] * (1.0 - 0.6 * f))))
    return qs, ns


def _bd(i, W):
    return max(0, (i - W) // BLOCK * BLOCK)


def work(c):
    qs, ns = _lengths(c)
    e, D, Hkv = SIZE[c["dtype"]], c["D"], c["Hkv"]
    row = (D + 4) if c["q8"] else D * e                      # one stored row
    T = sum(qs)
    if c["kind"] == "append":
        pools = 3 if c["rerope"] else 2
        n = T * (c["Hq"] + 2 * Hkv) * D * e + T * pools * Hkv * row + T * c["Hq"] * D * e * (pools - 1)
        if c["q8"]:
            n += pools * Hkv * (T * row + c["S"] * max(qs) * D * e)
        return {"bytes": float(n), "flops": float(T * 3 * (c["Hq"] + Hkv) * D)}
    if c["kind"] == "read":
        rows = sum(min(c["n"], n) for n in ns)
        return {"bytes": float(2 * Hkv * (rows * row + c["S"] * c["n"] * D * e)), "flops": float(2 * Hkv * rows * D)}
    W, MK, Hq = c["W"], c["M"] * c["K"], c["Hq"]
    n_bytes, keys = T * Hq * D * e * (3 if c["rerope"] else 2), 0
    for q, n in zip(qs, ns):
        i0, i1 = n - q, n - 1
        k1 = n - (max(0, i0 - W) if c["rerope"] else _bd(i0, W))
        k3 = max(0, max(0, i1 - W) - _bd(i0, W)) if c["rerope"] else 0
        n_bytes += Hkv * row * (k1 + k3 + n - _bd(i0, W))
        first, last = max(1, _bd(i0, W) // BLOCK), _bd(i1, W) // BLOCK
        n_bytes += max(0, last - first + 1) * Hkv * MK * (D * e + 4)
        for i in (range(i0, n) if q < 64 else ()):
            keys += i + 1 - _bd(i, W) + (MK if _bd(i, W) > 0 else 0)
        if q >= 64:
            for b in range(i0 // BLOCK, i1 // BLOCK + 1):
                lo, hi = max(i0, b * BLOCK), min(n, (b + 1) * BLOCK)
                keys += sum(range(lo + 1, hi + 1)) + (hi - lo) * ((MK if _bd(lo, W) > 0 else 0) - _bd(lo, W))
    if any(_bd(n - 1, W) > 0 for n in ns):
        n_bytes += Hkv * MK * D * e
    return {"bytes": float(n_bytes), "flops": 4.0 * D * Hq * keys}


# ------------------------------------------------------------------------------------------- inputs

def _angles(pos, D):
    inv = 1.0 / (BASE ** (torch.arange(0, D, 2, dtype=torch.float64, device=pos.device) / D))
    ang = pos.to(torch.float64)[..., None] * inv
    return ang.cos(), ang.sin()


def _rotate(x, pos):
    """fp32 rotation of x [..., H, D] to positions pos [...]: products and sum rounded one by one."""
    cos, sin = (t.float().unsqueeze(-2) for t in _angles(pos, x.shape[-1]))
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _quantise(x):
    """fp32 rows [..., D] -> int8 codes, fp32 scales [...]."""
    scale = x.abs().amax(-1) * (1.0 / 127.0)
    scale = torch.where(scale < 2.0 ** -126, torch.zeros_like(scale), scale)
    inv = torch.where(scale > 0, scale, torch.ones_like(scale)).reciprocal()
    return (torch.round(x * inv[..., None]) * (scale > 0)[..., None]).to(torch.int8), scale


def _fill(pool, scales, x, ids, q8):
    """Rows x [rows, Hkv, D] of consecutive positions into the pages ids."""
    P = pool.shape[2]
    pages = x.reshape(len(ids), P, *x.shape[1:]).transpose(1, 2)
    if q8:
        codes, sc = _quantise(pages.float())
        pool[ids], scales[ids] = codes, sc
    else:
        pool[ids] = pages.to(pool.dtype)


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)
    dt, q8, P, D, Hkv, S = DTYPES[c["dtype"]], c["q8"], c["P"], c["D"], c["Hkv"], c["S"]
    qs, ns = _lengths(c)
    T = sum(qs)
    # pages that hold rows this pass reads or writes: every sequence's from its first live row on
    if c["kind"] == "read":
        first = [max(0, n - c["n"]) for n in ns]
    elif c["kind"] == "append":
        first = [n - q for q, n in zip(qs, ns)]
    else:
        first = [_bd(n - q, c["W"]) for q, n in zip(qs, ns)]
    lo = [f // P for f in first]
    counts = [-(-n // P) - l for n, l in zip(ns, lo)]
    perm = torch.randperm(sum(counts), generator=g, device=dev).to(torch.int32)
    table = torch.full((S, -(-max(ns) // P)), -1, dtype=torch.int32, device=dev)
    at = 0
    for s in range(S):
        table[s, lo[s]: lo[s] + counts[s]] = perm[at: at + counts[s]]
        at += counts[s]
    npools = 3 if c.get("rerope", False) else 2               # k1, v (, k3); a read takes two pools
    shape = (sum(counts), Hkv, P, D)
    pools = [torch.zeros(shape, dtype=torch.int8 if q8 else dt, device=dev) for _ in range(npools)]
    scales = [torch.zeros(shape[:3], dtype=torch.float32, device=dev) if q8 else None for _ in range(npools)]
    st = dict(case=c, qs=qs, ns=ns, table=table, pools=pools, scales=scales,
              cu_q=torch.tensor([0] + qs, device=dev).cumsum(0).to(torch.int32), lens=torch.tensor(ns, dtype=torch.int32, device=dev))
    if c["kind"] == "append":
        st.update(q=rn(T, c["Hq"], D).to(dt), k=rn(T, Hkv, D).to(dt), v=rn(T, Hkv, D).to(dt),
                  starts=torch.tensor(first, dtype=torch.int32, device=dev), n=max(qs))
        return st
    for s in range(S):                                       # rows behind the end of a sequence: what an earlier owner left there
        ids = table[s, lo[s]: lo[s] + counts[s]].long()
        raw = rn(counts[s] * P, Hkv, D).to(dt)
        pos = torch.arange(lo[s] * P, (lo[s] + counts[s]) * P, device=dev)
        _fill(pools[0], scales[0], _rotate(raw, pos), ids, q8)
        _fill(pools[1], scales[1], rn(counts[s] * P, Hkv, D).to(dt), ids, q8)
        if npools == 3:
            _fill(pools[2], scales[2], raw, ids, q8)
    if c["kind"] == "read":
        st.update(starts=torch.tensor(first, dtype=torch.int32, device=dev), n=c["n"])
        return st
    W, MK, K = c["W"], c["M"] * c["K"], c["K"]
    pos = torch.cat([torch.arange(n - q, n, device=dev) for q, n in zip(qs, ns)])
    q = rn(T, c["Hq"], D)
    st["q1"] = _rotate(q, pos).to(dt)
    st["q2"] = _rotate(q, torch.full_like(pos, W + 1)).to(dt) if c["rerope"] else st["q1"]
    # snapshots: column (boundary block) % columns; as many columns as one sequence's chunk has boundaries
    blocks = [(_bd(n - q_, W) // BLOCK, _bd(n - 1, W) // BLOCK) for q_, n in zip(qs, ns)]
    cols = max(b1 - b0 + 1 for b0, b1 in blocks)
    snaps = torch.full((S, cols), -1, dtype=torch.int32, device=dev)
    older = []
    for s, (b0, b1) in enumerate(blocks):
        for b in range(max(1, b0), b1 + 1):
            snaps[s, b % cols] = len(older)
            older.append(b * BLOCK)
    st["snaps"], st["snap_host"], st["codebook"] = snaps, snaps.tolist(), None
    if older:
        cb = rn(Hkv, MK, D) * D ** -0.25
        mean = torch.tensor(older, dtype=torch.float32, device=dev).view(-1, 1, 1, 1) / K
        cnt = torch.floor(mean * torch.rand(len(older), Hkv, MK, 1, generator=g, device=dev) * 2.0 + 0.5)
        st.update(codebook=cb.to(dt), cnt=cnt[..., 0].contiguous(), vsum=(rn(len(older), Hkv, MK, D) * cnt.sqrt()).to(dt))
    return st


# ------------------------------------------------------------------------------------------- one pass

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from vqtree_b200 import api
    c, pools, scales = st["case"], st["pools"], st["scales"]
    two = [(pools[i], scales[i]) for i in range(len(pools))]
    if c["kind"] == "read":
        return api.paged_read(two, st["table"], st["starts"], st["lens"], st["n"], DTYPES[c["dtype"]])
    rerope = c["rerope"]
    pages = api.PagedKV(k1=pools[0], v=pools[1], k3=pools[2] if rerope else None, k1_scale=scales[0], v_scale=scales[1],
                        k3_scale=scales[2] if rerope else None)
    if c["kind"] == "append":
        q1, q2 = api.paged_append(st["k"], st["v"], pages, st["table"], st["cu_q"], st["lens"], q=st["q"],
                                  const_pos=c["W"] + 1 if rerope else None, base=BASE)
        back = api.paged_read(two, st["table"], st["starts"], st["lens"], st["n"], DTYPES[c["dtype"]]) if c["q8"] else pools
        return [q1] + ([q2] if rerope else []) + list(back)
    far = dict(codebook=st["codebook"], cnt=st["cnt"], vsum=st["vsum"], snap_table=st["snaps"]) if st["codebook"] is not None else {}
    return api.paged_attention(st["q1"], st["q2"], pages, st["table"], st["cu_q"], st["lens"], c["W"], max(st["qs"]), **far)


def _rows(pool, scale, ids, lo, hi):
    """Rows [lo, hi), counted from the first of the pages ids, as fp32 [Hkv, rows, D]."""
    x = pool[ids].float()
    if scale is not None:
        x = x * scale[ids][..., None]
    return x.transpose(1, 2).flatten(0, 1)[lo:hi].transpose(0, 1)


def _run_plain(st):
    c = st["case"]
    return {"append": _append_plain, "read": _read_plain, "attend": _attend_plain}[c["kind"]](st)


def _append_plain(st):
    c, table, P = st["case"], st["table"], st["case"]["P"]
    dt, dev = DTYPES[c["dtype"]], table.device
    seq = torch.cat([torch.full((q,), s, device=dev) for s, q in enumerate(st["qs"])])
    pos = torch.cat([torch.arange(n - q, n, device=dev) for q, n in zip(st["qs"], st["ns"])])
    page, row = table[seq, pos // P].long(), pos % P
    new = [_rotate(st["k"], pos), st["v"].float()] + ([st["k"].float()] if c["rerope"] else [])
    for pool, scale, x in zip(st["pools"], st["scales"], new):
        if c["q8"]:
            codes, sc = _quantise(x)
            pool[page, :, row], scale[page, :, row] = codes, sc
        else:
            pool[page, :, row] = x.to(dt)
    out = [_rotate(st["q"], pos).to(dt)]
    if c["rerope"]:
        out.append(_rotate(st["q"], torch.full_like(pos, c["W"] + 1)).to(dt))
    return out + (_read_plain(st) if c["q8"] else st["pools"])


def _read_plain(st):
    c, table, P = st["case"], st["table"], st["case"]["P"]
    r = torch.arange(st["n"], device=table.device)
    pos = st["starts"].long()[:, None] + r                                        # [S, n]
    valid = pos < st["lens"].long()[:, None]
    at = torch.where(valid, pos, st["starts"].long()[:, None])
    page = table.gather(1, at // P).long()
    out = []
    for pool, scale in zip(st["pools"], st["scales"]):
        x = pool[page, :, at % P].float()                                         # [S, n, Hkv, D]
        if scale is not None:
            x = x * scale[page, :, at % P][..., None]
        out.append((x * valid[..., None, None]).transpose(1, 2).to(DTYPES[c["dtype"]]).contiguous())
    return out


def _attend_plain(st):
    c = st["case"]
    W, P, D, Hkv, G = c["W"], c["P"], c["D"], c["Hkv"], c["Hq"] // c["Hkv"]
    table, pools, scales = st["table"], st["pools"], st["scales"]
    scale, dev = 1.0 / math.sqrt(D), table.device
    out = torch.empty_like(st["q1"])
    at = 0
    for s, (q, n) in enumerate(zip(st["qs"], st["ns"])):
        for blk in range((n - q) // BLOCK, (n - 1) // BLOCK + 1):                  # queries of one 128-block share a boundary
            i0, i1 = max(n - q, blk * BLOCK), min(n, (blk + 1) * BLOCK)
            b = _bd(i0, W)
            t = slice(at + i0 - (n - q), at + i1 - (n - q))
            i = torch.arange(i0, i1, device=dev)
            rows = lambda x: x[t].float().reshape(i1 - i0, Hkv, G, D).permute(1, 2, 0, 3)      # [Hkv, G, nq, D]
            ids = table[s, b // P: -(-i1 // P)].long()
            lo = b // P * P
            k1, v = (_rows(pools[x], scales[x], ids, b - lo, i1 - lo) for x in (0, 1))
            j = torch.arange(b, i1, device=dev)
            sc = rows(st["q1"]) @ k1[:, None].transpose(-1, -2) * scale
            if c["rerope"]:
                s2 = rows(st["q2"]) @ _rows(pools[2], scales[2], ids, b - lo, i1 - lo)[:, None].transpose(-1, -2) * scale
                sc = torch.where(j[None] < i[:, None] - W, s2, sc)
            sc = sc.masked_fill(j[None] > i[:, None], float("-inf"))
            m = sc.amax(-1, keepdim=True)
            if b > 0:
                mine = st["snap_host"][s]
                snap = mine[b // BLOCK % len(mine)]
                cnt, vsum = st["cnt"][snap], st["vsum"][snap].float()
                sf = rows(st["q2"]) @ st["codebook"].float()[:, None].transpose(-1, -2) * scale
                sf = sf.masked_fill((cnt <= 0)[:, None, None], float("-inf"))
                m = torch.maximum(m, sf.amax(-1, keepdim=True))
            p = torch.exp(sc - m)
            num, den = p @ v[:, None], p.sum(-1)
            if b > 0:
                p = torch.exp(sf - m)
                num, den = num + p @ vsum[:, None], den + (p * cnt[:, None, None]).sum(-1)
            out[t] = (num / den[..., None]).permute(2, 0, 1, 3).reshape(i1 - i0, Hkv * G, D).to(out.dtype)
        at += q
    return out


# ------------------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["kind"] == "attend":
        return _attend_exact(st)
    P, dev = c["P"], st["table"].device
    table, f64 = st["table"].cpu().tolist(), torch.float64

    def turned(x, pos):                                                           # complex product instead of two half rows
        D = x.shape[-1]
        x = x.to(f64)
        cos, sin = _angles(pos, D)
        z = torch.complex(x[..., : D // 2], x[..., D // 2:]) * torch.complex(cos, sin)[:, None]
        return torch.cat((z.real, z.imag), -1)

    def held(x):                                                                  # what an 8-bit row stands for
        s = x.abs().amax(-1, keepdim=True) / 127
        return torch.where(s > 0, torch.round(x / s) * s, torch.zeros_like(x))

    def back(rows_of):                                                            # dense rows of every sequence
        out = torch.zeros(c["S"], c["Hkv"], st["n"], c["D"], dtype=f64, device=dev)
        for s, n in enumerate(st["ns"]):
            f = int(st["starts"][s])
            m = min(st["n"], n - f)
            out[s, :, :m] = rows_of(s, f, f + m).transpose(0, 1)
        return out

    if c["kind"] == "read":
        res = []
        for pool, scale in zip(st["pools"], st["scales"]):
            flat = pool.to(f64) * (1.0 if scale is None else scale.to(f64)[..., None])
            res.append(back(lambda s, a, b: torch.stack([flat[table[s][j // P], :, j % P] for j in range(a, b)])
                            if b - a < 300 else flat[st["table"][s].long().clamp(min=0)].transpose(1, 2).flatten(0, 1)[a:b]))
        return res
    pos = torch.cat([torch.arange(n - q, n, device=dev) for q, n in zip(st["qs"], st["ns"])])
    new = [turned(st["k"], pos), st["v"].to(f64)] + ([st["k"].to(f64)] if c["rerope"] else [])
    res = [turned(st["q"], pos)] + ([turned(st["q"], torch.full_like(pos, c["W"] + 1))] if c["rerope"] else [])
    start = [sum(st["qs"][:s]) for s in range(c["S"])]
    if c["q8"]:
        new = [held(x) for x in new]
        return res + [back(lambda s, a, b, x=x: x[start[s]: start[s] + b - a]) for x in new]
    for pool, x in zip(st["pools"], new):
        pool = pool.to(f64)
        for s, (q, n) in enumerate(zip(st["qs"], st["ns"])):
            for page in range((n - q) // P, (n - 1) // P + 1):
                a, b = max(n - q, page * P), min(n, (page + 1) * P)
                pool[table[s][page], :, a - page * P: b - page * P] = x[start[s] + a - (n - q): start[s] + b - (n - q)].transpose(0, 1)
        res.append(pool)
    return res


def _attend_exact(st):
    """Every sequence and head by itself: one weight matrix over all its live keys and the codes of each boundary."""
    c = st["case"]
    W, P, D, G = c["W"], c["P"], c["D"], c["Hq"] // c["Hkv"]
    f64, dev = torch.float64, st["table"].device
    if work(c)["flops"] > 4.0e11:
        return None
    out, at = torch.zeros(st["q1"].shape, dtype=f64, device=dev), 0
    for s, (q, n) in enumerate(zip(st["qs"], st["ns"])):
        first = (n - q - W) // BLOCK * BLOCK if n - q > W else 0
        ids, skip = st["table"][s, first // P: (n + P - 1) // P].long(), first % P
        live = []
        for pool, sc in zip(st["pools"], st["scales"]):
            x = pool[ids].to(f64)
            x = x if sc is None else x * sc[ids].to(f64).unsqueeze(-1)
            live.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, skip: skip + n - first])
        i = torch.arange(n - q, n, device=dev).view(-1, 1)
        j = torch.arange(first, n, device=dev).view(1, -1)
        bound = ((i - W).clamp(min=0) // BLOCK) * BLOCK
        near, far_exact = (j <= i) & (j >= i - W), (j < i - W) & (j >= bound)
        for h in range(c["Hq"]):
            a, b2 = st["q1"][at: at + q, h].to(f64), st["q2"][at: at + q, h].to(f64)
            k1, v, k3 = live[0][h // G], live[1][h // G], live[2 if c["rerope"] else 0][h // G]
            score = torch.where(near, a @ k1.T, torch.where(far_exact, b2 @ k3.T, torch.full((), -math.inf, dtype=f64, device=dev))) / math.sqrt(D)
            top = score.max(1).values
            sums = {}
            for b in sorted(set(bound.flatten().tolist()) - {0}) if st["codebook"] is not None else []:
                mine = (bound == b).flatten()
                k = int(st["snaps"][s, (b // BLOCK) % st["snaps"].shape[1]])
                cnt = st["cnt"][k, h // G].to(f64)
                e = b2[mine] @ st["codebook"][h // G].to(f64).T / math.sqrt(D)
                e = torch.where(cnt > 0, e, torch.full((), -math.inf, dtype=f64, device=dev))
                top[mine] = torch.maximum(top[mine], e.max(1).values)
                sums[b] = (mine, e, cnt, st["vsum"][k, h // G].to(f64))
            weight = (score - top[:, None]).exp()
            num, den = weight @ v, weight.sum(1)
            for mine, e, cnt, vs in sums.values():
                weight = (e - top[mine, None]).exp()
                num[mine] += weight @ vs
                den[mine] += weight @ cnt
            out[at: at + q, h] = num / den[:, None]
        at += q
    return out
