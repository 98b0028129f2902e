"""Plain CPU forms of the paged entry points of ``vqtree_b200.api`` (test infrastructure): the host logic of the paged cache runs on them
without a GPU."""
from __future__ import annotations

import contextlib
import math

import torch

from tests import fake_backend
from tests.paged_cases import boundary, quantise32, rotate64


def _rows(cu_q, lens):
    for s in range(len(lens)):
        t0, q, n = int(cu_q[s]), int(cu_q[s + 1] - cu_q[s]), int(lens[s])
        for x in range(q):
            yield s, t0 + x, n - q + x


def paged_append(k, v, pages, block_table, cu_q, seq_lens, q=None, const_pos=None, rotate=True, base=10000.0, n_pos=None):
    P = pages.k1.shape[2]
    q1 = torch.empty_like(q) if q is not None else None
    q2 = torch.empty_like(q) if q is not None and const_pos is not None else None
    for s, t, pos in _rows(cu_q, seq_lens):
        page, r = int(block_table[s, pos // P]), pos % P
        assert 0 <= page < pages.k1.shape[0], "no page"
        turn = lambda x, i: rotate64(x[None], torch.tensor([i]), base)[0].float() if rotate else x.float()
        for pool, scale, x in ((pages.k1, pages.k1_scale, turn(k[t], pos)), (pages.v, pages.v_scale, v[t].float()), (pages.k3, pages.k3_scale, k[t].float())):
            if pool is None:
                continue
            if scale is None:
                pool[page, :, r] = x.to(pool.dtype)
            else:
                pool[page, :, r], scale[page, :, r] = quantise32(x)
        if q1 is not None:
            q1[t] = turn(q[t], pos).to(q.dtype)
        if q2 is not None:
            q2[t] = turn(q[t], const_pos).to(q.dtype)
    return q1, q2


def paged_read(pools, block_table, starts, seq_lens, n, out_dtype=None):
    outs = []
    for pool, scale in pools:
        P = pool.shape[2]
        out = torch.zeros(block_table.shape[0], pool.shape[1], n, pool.shape[3], dtype=out_dtype or pool.dtype)
        for s in range(block_table.shape[0]):
            pos = int(starts[s]) + torch.arange(n)
            r = ((pos >= 0) & (pos < int(seq_lens[s]))).nonzero()[:, 0]
            page = block_table[s, pos[r] // P].long()
            assert (page >= 0).all(), "no page"
            x = pool[page, :, pos[r] % P].double()
            out[s, :, r] = (x if scale is None else x * scale[page, :, pos[r] % P].double()[..., None]).transpose(0, 1).to(out.dtype)
        outs.append(out)
    return outs


def paged_attention(q1, q2, pages, block_table, cu_q, seq_lens, window, max_q, codebook=None, cnt=None, vsum=None, snap_table=None, scale=None,
                    out=None):
    P, Hkv, D = pages.k1.shape[2], pages.k1.shape[1], pages.k1.shape[3]
    G = q1.shape[1] // Hkv
    out = torch.empty_like(q1) if out is None else out
    sc = scale or 1.0 / math.sqrt(D)
    for s, t, i in _rows(cu_q, seq_lens):
        b = boundary(i, window)
        a1, a2 = (x[t].double().reshape(Hkv, G, D) for x in (q1, q2))
        j = torch.arange(b, i + 1)
        page, r = block_table[s, j // P].long(), j % P
        assert (page >= 0).all(), "no page"
        held = lambda pool, scale: pool[page, :, r].double() * (1.0 if scale is None else scale[page, :, r].double()[..., None])   # [J, Hkv, D]
        scores, vals, w = torch.einsum("hgd,jhd->hgj", a1, held(pages.k1, pages.k1_scale)) * sc, held(pages.v, pages.v_scale).transpose(0, 1), torch.ones(Hkv, len(j))
        if pages.k3 is not None:
            scores = torch.where(j < i - window, torch.einsum("hgd,jhd->hgj", a2, held(pages.k3, pages.k3_scale)) * sc, scores)
        if b > 0 and codebook is not None:
            k = int(snap_table[s, b // 128 % snap_table.shape[1]])
            assert k >= 0, "no snapshot"
            far = (torch.einsum("hgd,hrd->hgr", a2, codebook.double()) * sc).masked_fill((cnt[k] == 0)[:, None], -math.inf)
            scores, vals, w = torch.cat((scores, far), -1), torch.cat((vals, vsum[k].double()), 1), torch.cat((w, cnt[k]), 1)
        w = w.double()
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        out[t] = (torch.einsum("hgj,hjd->hgd", p, vals) / (p * w[:, None]).sum(-1, keepdim=True)).reshape(Hkv * G, D).to(out.dtype)
    return out


@contextlib.contextmanager
def installed():
    from vqtree_b200 import api
    names = ("paged_append", "paged_read", "paged_attention")
    saved = {n: getattr(api, n) for n in names}
    with fake_backend.installed():
        try:
            for n in names:
                setattr(api, n, globals()[n])
            yield
        finally:
            for n, f in saved.items():
                setattr(api, n, f)
