"""Small paged caches with everything that can go wrong in them, and a plain 64-bit implementation of their operators (CPU)."""
from __future__ import annotations

import math

import torch

BLOCK = 128


def boundary(i, W):
    return max(0, (i - W) // BLOCK * BLOCK)


def rotate64(x, pos, base=10000.0):
    """x [..., H, D] rotated to positions pos [...] in the half-split convention, float64."""
    D = x.shape[-1]
    inv = base ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = pos.double()[..., None] * inv
    c, s = ang.cos()[..., None, :], ang.sin()[..., None, :]
    a, b = x.double().split(D // 2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def quantise32(x):
    """The documented 8-bit rows: x [..., D] fp32 -> (int8 codes, fp32 scales), every operation rounded to fp32."""
    x = x.float()
    finite = torch.isfinite(x).all(-1)
    scale = torch.where(finite, x.abs().amax(-1), torch.zeros(())) * torch.tensor(1.0 / 127.0, dtype=torch.float32)
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, torch.zeros(()), scale)
    inv = torch.where(scale > 0, scale, torch.ones(())).reciprocal() * (scale > 0)
    codes = torch.where(finite[..., None], torch.round(x * inv[..., None]), torch.zeros(())).to(torch.int8)
    return codes, torch.where(finite, scale, torch.full((), float("nan")))


class Case:
    """Sequences of ``lens`` tokens, the last ``qs`` of them new.  CPU tensors; ``to_gpu`` gives what the entry points take."""

    def __init__(self, seed, qs, lens, Hkv, G, D, P, W, MK=128, dtype=torch.bfloat16, q8=False, rerope=True, far=True, tail=0, free=True,
                 cols=None, garbage=True, scale_v=1.0):
        g = torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g)
        self.qs, self.lens, self.Hkv, self.G, self.D, self.P, self.W, self.MK = list(qs), list(lens), Hkv, G, D, P, W, MK
        self.dtype, self.q8, self.rerope, self.tail = dtype, q8, rerope, tail
        S, T = len(qs), sum(qs)
        self.S, self.T = S, T
        MB = max(1, -(-max(lens) // P))
        # pages of live rows only, in a shuffled pool with one page that nobody owns
        need = [(s, c) for s in range(S) for c in range((boundary(lens[s] - qs[s], W) if free and qs[s] else 0) // P, -(-lens[s] // P))]
        perm = torch.randperm(len(need) + 1, generator=g)
        self.table = torch.full((S, MB), -1, dtype=torch.int32)
        for (s, c), pg in zip(need, perm):
            self.table[s, c] = pg
        NP = len(need) + 1
        self.dense = []                                    # per sequence: k1, k3, v float64 [n, Hkv, D] as the pools hold them
        act = lambda x: x.to(dtype)
        pools = [torch.full((NP, Hkv, P, D), float("nan") if garbage and not q8 else 0.0).to(torch.int8 if q8 else dtype) for _ in range(3)]
        if q8 and garbage:
            pools = [torch.randint(-128, 128, p.shape, generator=g, dtype=torch.int8) for p in pools]
        scales = [torch.full((NP, Hkv, P), float("nan") if garbage else 0.0) for _ in range(3)] if q8 else [None] * 3
        for s in range(S):
            n = lens[s]
            raw, v = rn(n, Hkv, D), rn(n, Hkv, D) * scale_v
            k1 = rotate64(raw, torch.arange(n)).float()
            held = []
            for i, x in enumerate((k1, raw, v)):
                if q8:
                    codes, sc = quantise32(x)
                    val = codes.double() * sc.double()[..., None]
                else:
                    codes, sc, val = act(x), None, act(x).double()
                held.append(val)
                for c in range(MB):
                    pg = int(self.table[s, c])
                    if pg >= 0:
                        m = min(P, n - c * P)
                        pools[i][pg, :, :m] = codes[c * P: c * P + m].transpose(0, 1)
                        if q8:
                            scales[i][pg, :, :m] = sc[c * P: c * P + m].T
            self.dense.append(held)
        self.pools, self.scales = pools, scales
        q = rn(T + tail, Hkv * G, D)
        self.pos = torch.cat([torch.arange(n - q_, n) for q_, n in zip(qs, lens)] + [torch.zeros(tail, dtype=torch.long)])
        self.q1 = act(rotate64(q, self.pos).float())
        self.q2 = act(rotate64(q, torch.full_like(self.pos, W + 1)).float()) if rerope else self.q1
        self.cu_q = torch.tensor([0] + self.qs).cumsum(0).to(torch.int32)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32)
        # snapshots
        spans = [(boundary(n - q_, W) // BLOCK, boundary(n - 1, W) // BLOCK) if q_ else (0, 0) for q_, n in zip(qs, lens)]
        self.cols = cols or max(b1 - b0 + 1 for b0, b1 in spans)
        ids = [(s, b) for s, (b0, b1) in enumerate(spans) for b in range(max(1, b0), b1 + 1)]
        self.far = far and bool(ids)
        self.snap_table = torch.full((S, self.cols), -1, dtype=torch.int32)
        if self.far:
            NS = len(ids) + 1
            perm = torch.randperm(NS, generator=g)
            for (s, b), k in zip(ids, perm):
                self.snap_table[s, b % self.cols] = k
            self.cb = act(rn(Hkv, MK, D) * D ** -0.25)
            self.cnt = torch.randint(0, 6, (NS, Hkv, MK), generator=g).float()
            self.cnt[:, :, ::7] = 0
            self.vsum = act(rn(NS, Hkv, MK, D) * self.cnt.sqrt()[..., None] * scale_v)

    def pages(self, dev="cuda", layout=None):
        from vqtree_b200 import api
        put = (lambda t: t.to(dev)) if layout is None else (lambda t: layout(t.to(dev)))
        t = [put(p) for p in self.pools]
        s = [x.to(dev) if x is not None else None for x in self.scales]
        return api.PagedKV(t[0], t[2], t[1] if self.rerope else None, s[0], s[2], s[1] if self.rerope else None)

    def far_args(self, dev="cuda"):
        if not self.far:
            return {}
        return dict(codebook=self.cb.to(dev), cnt=self.cnt.to(dev), vsum=self.vsum.to(dev), snap_table=self.snap_table.to(dev))

    def attend(self, api, pages=None, out=None, **kw):
        d = lambda t: t.cuda()
        q1 = d(self.q1)
        q2 = d(self.q2) if self.rerope else q1
        return api.paged_attention(q1, q2, pages or self.pages(), d(self.table), d(self.cu_q), d(self.seq_lens), self.W, kw.pop("max_q", max(self.qs)),
                                   out=out, **self.far_args(), **kw)

    def expected(self, scale=None):
        """(attention of every new token, sums of |weight * value| / denominator), float64 [T, Hq, D]."""
        W, G, D, Hkv = self.W, self.G, self.D, self.Hkv
        sc = scale or 1.0 / math.sqrt(D)
        out = torch.zeros(self.T, Hkv * G, D, dtype=torch.float64)
        mag = torch.zeros_like(out)
        t = 0
        for s in range(self.S):
            k1, k3, v = self.dense[s]
            for i in range(self.lens[s] - self.qs[s], self.lens[s]):
                b = boundary(i, W)
                q1, q2 = (x[t].double().reshape(Hkv, G, D) for x in (self.q1, self.q2))
                near = max(0, i - W) if self.rerope else b
                score = torch.cat((torch.einsum("hgd,jhd->hgj", q2, k3[b:near]), torch.einsum("hgd,jhd->hgj", q1, k1[near:i + 1])), -1) * sc
                vals, w = v[b:i + 1].transpose(0, 1), torch.ones(Hkv, i + 1 - b, dtype=torch.float64)
                if self.far and b > 0:
                    k = int(self.snap_table[s, b // BLOCK % self.cols])
                    f = torch.einsum("hgd,hrd->hgr", q2, self.cb.double()) * sc
                    f = f.masked_fill((self.cnt[k] == 0)[:, None], -math.inf)
                    score, w = torch.cat((f, score), -1), torch.cat((self.cnt[k].double(), w), 1)
                    vals = torch.cat((self.vsum[k].double(), vals), 1)
                p = (score - score.amax(-1, keepdim=True)).exp()
                den = (p * w[:, None]).sum(-1, keepdim=True)
                out[t] = (torch.einsum("hgj,hjd->hgd", p, vals) / den).reshape(Hkv * G, D)
                mag[t] = (torch.einsum("hgj,hjd->hgd", p, vals.abs()) / den).reshape(Hkv * G, D)
                t += 1
        return out, mag

    def tolerance(self, ref, mag):
        """What rounding allows, element by element.  The output is rounded once (u |ref|, u half a step) and every weight once before it
        meets its value row (u per term: u mag).  fp32: scores are sums of D products, |s| below 16 here, so a weight is off by
        (D + 32) 2^-24 * 16 at most relative to itself in numerator and denominator each, and sums of up to 4096 terms lose 2^-12 of
        mag at the worst and 2^-18 as they are added here (64 lanes and warps); half: weights below 2^-14 of the largest are off by 2^-25."""
        u = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[self.dtype]
        fp32 = 2 * (self.D + 32) * 16 * 2.0 ** -24 + 2.0 ** -18
        small = 2.0 ** -25 * 4096 * (mag.amax() if self.dtype == torch.float16 else 0.0)
        return u * ref.abs() + (u + fp32) * mag + small + 1e-30


def check_attention(got, case):
    ref, mag = case.expected()
    got = got[:case.T].double().cpu()
    tol = case.tolerance(ref, mag)
    err = (got - ref).abs()
    assert torch.isfinite(got).all(), f"{int((~torch.isfinite(got)).sum())} values are not finite"
    worst = float((err / tol).max())
    assert worst <= 1.0, f"error is {worst:.2f} of what rounding allows (max {float(err.max()):.3e})"
