"""Runs of a paged cache as a server makes them, on either device: sequences that come and go, chunks of every size."""
from __future__ import annotations

import numpy as np
import torch

from oracle import vq_oracle as vo
from tests.vq_cases import make_case, oracle_prefill
from vqtree_b200.paged_cache import PagedVectorQuantizedCache


def whole_sequences(lens, Hq, Hkv, D, M, K, W, dtype, rerope=True):
    """Raw q, k, v per sequence, a shared codebook, and every row's result by the naive per-query loop of the oracle."""
    cases, want = [], []
    g = torch.Generator().manual_seed(sum(lens))
    cb = torch.randn(Hkv, M, K, D, generator=g) * D ** -0.25
    for n in lens:
        q, k, v = (torch.randn(n, h, D, generator=g).to(dtype) for h in (Hq, Hkv, Hkv))
        cos, sin = vo.rope_tables(max(n, W + 2), D)
        f = lambda t: t.float().transpose(0, 1)[None].numpy()
        rnd = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dtype).float().numpy()
        q1, k1 = rnd(vo.apply_rope(f(q), cos, sin, np.arange(n))), rnd(vo.apply_rope(f(k), cos, sin, np.arange(n)))
        q2, k3 = (rnd(vo.apply_rope(f(q), cos, sin, np.full(n, W + 1))), f(k)) if rerope else (q1, k1)
        codes = vo.assign_codes(k3, cb.numpy())
        cb_act = cb.to(dtype).float().numpy()
        out = vo.attn_naive(q1, q2, k1, k3, f(v), cb_act, codes, W, None)[0]
        cases.append((q, k, v))
        want.append(torch.from_numpy(out).transpose(0, 1))                   # [n, Hq, D]
    return cb, cases, want


def serve(cases, cb, schedule, W, dtype, device, *, quantized=False, rerope=True, page_size=32, num_pages=64, max_sequences=4, **kw):
    """schedule: per call a dict {sequence number: new tokens}.  Returns per sequence the rows in order, and the cache."""
    cache = PagedVectorQuantizedCache(W, cb, num_pages, max_sequences, page_size=page_size, dtype=dtype, quantized=quantized, rerope=rerope, device=device,
                                      max_length=2048, **kw)
    got, sids, at = {i: [] for i in range(len(cases))}, {}, {i: 0 for i in range(len(cases))}
    for call in schedule:
        for i in call:
            if i not in sids:
                sids[i] = cache.add_sequence()
        parts = [[x[at[i]: at[i] + m] for x in cases[i]] for i, m in call.items()]
        q, k, v = (torch.cat([p[j] for p in parts]).to(device) for j in range(3))
        out = cache.attend([sids[i] for i in call], list(call.values()), q, k, v).view(q.shape)
        for (i, m), rows in zip(call.items(), out.split(list(call.values()))):
            got[i].append(rows.float().cpu())
            at[i] += m
    return {i: torch.cat(r) for i, r in got.items() if r}, cache, sids
