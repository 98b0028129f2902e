"""A serving cache over the paged operators: many sequences of different lengths, tokens in chunks of any size.

``VectorQuantizedReRoPECache`` (attn_vq.py) holds one length per batch and takes a prompt or one token at a time, like the reference's cache
(ops/attn_vq.py:31-173, "Only support prefilling or generation").  ``PagedVectorQuantizedCache`` holds one attention layer of up to
``max_sequences`` sequences: window rows in pages of a shared pool (16 or 8 bits), counts and value sums per code of everything older,
and one call - ``attend`` - that takes any mixture of prompts, pieces of prompts, second turns, drafted tokens and single tokens.  Every row of
its result is what that row of a prefill over the whole sequence is defined to be; with 8-bit pages the window's keys and values, and
the keys that are quantised into codes, are those the pages stand for.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence

import torch

from . import api
from .attn_vq import BLOCK_SIZE, VectorQuantizedReRoPECache


class OutOfPages(RuntimeError):
    """The pool (or the spare snapshots) cannot hold what the call brings; nothing has been changed."""


class _Sequence:
    __slots__ = ("slot", "n", "bd", "first", "pages")

    def __init__(self, slot: int):
        self.slot, self.n, self.bd = slot, 0, 0
        self.first = 0                 # page column of pages[0]
        self.pages: List[int] = []     # pages of columns first, first + 1, ...


def _runs(numbers) -> List[slice]:
    """Slices of neighbouring numbers: few large copies instead of many."""
    out = []
    for x in sorted(numbers):
        if out and out[-1].stop == x:
            out[-1] = slice(out[-1].start, x + 1)
        else:
            out.append(slice(x, x + 1))
    return out


class PagedVectorQuantizedCache:
    """window_length, codebook ([H,C,D] or [H,M,K,D]), rope_base: as VectorQuantizedReRoPECache.  num_pages pages of page_size (16, 32, 64
    or 128) tokens are shared by the sequences; a sequence needs those of its window, up to window + 128 tokens and the chunk in flight.
    quantized: 8-bit pages.  rerope False: plain rotary positions (no raw keys; the rotated keys are quantised into codes).
    spare_snapshots: copies of the value sums a call may need beyond one per sequence (a chunk of c tokens: c / 128 + 1).
    Calls of one cache belong on one stream."""

    def __init__(self, window_length: int, codebook: torch.Tensor, num_pages: int, max_sequences: int, *, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, quantized: bool = False, rerope: bool = True, rope_base: Optional[float] = None,
                 max_length: int = 1 << 17, spare_snapshots: int = 32, device="cuda"):
        assert window_length % BLOCK_SIZE == 0 and window_length > 0
        assert page_size in (16, 32, 64, 128), "pages of 16, 32, 64 or 128 tokens"
        assert max_length % page_size == 0 and max_length >= window_length
        self.window_length, self.page_size, self.max_length = window_length, page_size, max_length
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:      # the current one now, not that of a later call
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.codebooks = (codebook if codebook.dim() == 4 else codebook[:, None]).to(self.device, torch.float32).contiguous()   # [H,M,K,D]
        H, M, K, D = self.codebooks.shape
        assert M * K % BLOCK_SIZE == 0
        self.codebook_act = self.codebooks.reshape(H, M * K, D).to(dtype).contiguous()
        self.dtype, self.rerope, self.rope_base = dtype, rerope, rope_base or 10000.0
        self.pages = api.PagedKV.allocate(num_pages, H, page_size, D, torch.int8 if quantized else dtype, self.device, raw_keys=rerope)
        self.block_table = torch.full((max_sequences, max_length // page_size), -1, dtype=torch.int32, device=self.device)
        # running aggregates: row = slot of the sequence; the rows behind them are copies for chunks that span boundaries
        self.max_sequences, self.spare = max_sequences, spare_snapshots
        rows = max_sequences + spare_snapshots
        self.cnt = torch.zeros(rows, H, M * K, dtype=torch.float32, device=self.device)
        self.vsum32 = torch.zeros(max_sequences, H, M * K, D, dtype=torch.float32, device=self.device)
        self.vsum = torch.zeros(rows, H, M * K, D, dtype=dtype, device=self.device)
        self._free_pages = list(range(num_pages - 1, -1, -1))
        self._free_slots = list(range(max_sequences - 1, -1, -1))
        self._sequences = {}
        self._next_id = 0

    # ---- sequences
    def add_sequence(self) -> int:
        """A new, empty sequence; returns its id."""
        if not self._free_slots:
            raise OutOfPages("every sequence slot is taken")
        seq = _Sequence(self._free_slots.pop())
        self.cnt[seq.slot].zero_()
        self.vsum32[seq.slot].zero_()
        self.vsum[seq.slot].zero_()
        sid, self._next_id = self._next_id, self._next_id + 1
        self._sequences[sid] = seq
        return sid

    def remove_sequence(self, sid: int) -> None:
        seq = self._sequences.pop(sid)
        self._free_pages.extend(reversed(seq.pages))
        self._free_slots.append(seq.slot)

    def length(self, sid: int) -> int:
        return self._sequences[sid].n

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    def _boundary(self, i: int) -> int:
        return max(0, (i - self.window_length) // BLOCK_SIZE * BLOCK_SIZE)

    # ---- the call
    def attend(self, sids: Sequence[int], q_lens: Sequence[int], query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
               scale: Optional[float] = None) -> torch.Tensor:
        """query [T,Hq,D], key, value [T,Hkv,D] un-rotated: q_lens[i] new tokens of sequence sids[i], packed one after another.
        Returns [T, Hq*D]."""
        sids, q_lens = list(sids), [int(x) for x in q_lens]
        T, hq, d = query.shape
        if len(sids) != len(q_lens) or len(set(sids)) != len(sids):
            raise ValueError("one length per sequence, every sequence once")
        if min(q_lens, default=0) < 0 or sum(q_lens) != T:
            raise ValueError("q_lens must add up to the rows of query")
        if query.dtype != self.dtype:
            raise ValueError(f"the cache holds {self.dtype}")
        if key.shape != value.shape or tuple(key.shape) != (T, self.codebooks.shape[0], d) or d != self.codebooks.shape[3]:
            raise ValueError("key and value must be [T, kv heads, head dim] of the codebook")
        if key.dtype != self.dtype or value.dtype != self.dtype:
            raise ValueError(f"the cache holds {self.dtype}")
        if hq % key.shape[1] != 0 or not 1 <= hq // key.shape[1] <= 128:
            raise ValueError("query heads must be 1 to 128 times the kv heads")
        if T == 0:
            return query.new_empty(0, hq * d)
        seqs = [self._sequences[s] for s in sids]
        before, saved = [(seq, seq.bd, len(seq.pages)) for seq in seqs], []
        try:
            lens, out = self._run(seqs, q_lens, query, key, value, scale, saved)
        except BaseException:                               # out of memory, say: the sequences stay what they were before the call
            self._undo(before, saved)
            raise
        for seq, n in zip(seqs, lens):                      # pages in front of the boundary have become counts and sums
            seq.n = n
            gone = seq.bd // self.page_size - seq.first
            if gone > 0:
                self._free_pages.extend(reversed(seq.pages[:gone]))
                del seq.pages[:gone]
                seq.first += gone
        return out.reshape(T, hq * d)

    def _run(self, seqs, q_lens, query, key, value, scale, saved):
        """The call on checked arguments: what it changes, but for ``n`` and the pages that fall free, ``_undo`` takes back."""
        lens = self._reserve(seqs, q_lens)
        meta = [0]
        for x in q_lens:
            meta.append(meta[-1] + x)
        S = len(seqs)
        meta = self._upload(meta + lens + [s.slot for s in seqs])
        cu_q, seq_lens, slots = meta[: S + 1], meta[S + 1: 2 * S + 1], meta[2 * S + 1:]
        table = self.block_table.index_select(0, slots)
        W = self.window_length
        q1, q2 = api.paged_append(key, value, self.pages, table, cu_q, seq_lens, q=query, const_pos=W + 1 if self.rerope else None,
                                  base=self.rope_base, n_pos=max(self.max_length, W + 2))
        snaps = self._fold(seqs, q_lens, table, seq_lens, saved)
        out = api.paged_attention(q1, q2 if self.rerope else q1, self.pages, table, cu_q, seq_lens, W, max(q_lens), codebook=self.codebook_act,
                                  cnt=self.cnt, vsum=self.vsum, snap_table=snaps, scale=scale or 1.0 / math.sqrt(query.shape[2]))
        return lens, out

    def _undo(self, before, saved) -> None:
        """After a call that failed: pages it took go back, boundaries and aggregates are those of before."""
        for seq, bd, pages in before:
            self._free_pages.extend(reversed(seq.pages[pages:]))
            del seq.pages[pages:]
            seq.bd = bd
        for slots, cnt, vsum32 in saved:
            self.cnt[slots].copy_(cnt)
            self.vsum32[slots].copy_(vsum32)
            self.vsum[slots].copy_(vsum32)

    def _upload(self, numbers) -> torch.Tensor:
        t = torch.tensor(numbers, dtype=torch.int32)
        return t.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else t

    def _reserve(self, seqs, q_lens) -> List[int]:
        """Pages for the new tokens; all or nothing.  Returns the lengths with them."""
        P, lens, want, copies = self.page_size, [], [], 0
        for seq, q in zip(seqs, q_lens):
            n = seq.n + q
            if n > self.max_length:
                raise ValueError(f"a sequence of {n} tokens exceeds max_length")
            lens.append(n)
            want.append(-(-n // P) - seq.first - len(seq.pages))
            if q:
                copies += (self._boundary(n - 1) - max(seq.bd, self._boundary(seq.n))) // BLOCK_SIZE
        if sum(want) > len(self._free_pages):
            raise OutOfPages(f"{sum(want)} pages wanted, {len(self._free_pages)} free")
        if copies > self.spare:
            raise OutOfPages(f"{copies} snapshots wanted, {self.spare} spare")
        where, what = [], []
        cols = self.block_table.shape[1]
        for seq, w in zip(seqs, want):
            for _ in range(w):
                where.append(seq.slot * cols + seq.first + len(seq.pages))
                seq.pages.append(self._free_pages.pop())
                what.append(seq.pages[-1])
        if where:
            new = self._upload(where + what)
            self.block_table.view(-1).index_copy_(0, new[: len(where)].long(), new[len(where):])
        return lens

    def _fold(self, seqs, q_lens, table, seq_lens, saved) -> torch.Tensor:
        """Blocks that the new queries no longer see one by one go into counts and value sums; where the queries of one call have
        several boundaries, the aggregates of the earlier ones are kept in spare rows.  Returns the snapshot table of the call.
        saved: takes (slots, counts, fp32 sums) of the sequences that change, as they were."""
        leaving = []                                        # (index of the sequence in the call, block)
        plan = []
        for x, (seq, q) in enumerate(zip(seqs, q_lens)):
            b0 = self._boundary(seq.n) if q else seq.bd
            b1 = self._boundary(seq.n + q - 1) if q else seq.bd
            plan.append((b0, b1))
            leaving += [(x, b) for b in range(seq.bd, b1, BLOCK_SIZE)]
        cols = max((b1 - b0) // BLOCK_SIZE + 1 for b0, b1 in plan)
        snaps = [[-1] * cols for _ in seqs]
        if leaving:
            kv = self.pages
            pair = [(kv.k3, kv.k3_scale) if self.rerope else (kv.k1, kv.k1_scale), (kv.v, kv.v_scale)]
            idx = self._upload([x for x, _ in leaving] + [b for _, b in leaving])
            which, starts = idx[: len(leaving)], idx[len(leaving):]
            raw, val = api.paged_read(pair, table.index_select(0, which), starts, seq_lens.index_select(0, which), BLOCK_SIZE, self.dtype)
            codes = api.assign_codes(raw, self.codebooks)
            for slots in _runs({seqs[x].slot for x, _ in leaving}):
                saved.append((slots, self.cnt[slots].clone(), self.vsum32[slots].clone()))
        K, spare, at = self.codebooks.shape[2], self.max_sequences, 0
        for x, (seq, (b0, b1)) in enumerate(zip(seqs, plan)):
            s = seq.slot
            for b in range(seq.bd, b1, BLOCK_SIZE):
                if b >= b0:                                 # queries of this call stand at boundary b
                    self.cnt[spare].copy_(self.cnt[s])
                    self.vsum[spare].copy_(self.vsum[s])
                    snaps[x][b // BLOCK_SIZE % cols] = spare
                    spare += 1
                api.cache_advance(codes[at: at + 1], val[at: at + 1], K, self.cnt[s: s + 1], self.vsum32[s: s + 1],
                                  self.vsum[s: s + 1] if self.dtype != torch.float32 else None)
                if self.dtype == torch.float32:
                    self.vsum[s].copy_(self.vsum32[s])
                at += 1
            seq.bd = b1
            snaps[x][b1 // BLOCK_SIZE % cols] = s
        return self._upload([e for row in snaps for e in row]).view(len(seqs), cols)

    # ---- to and from the dense cache
    def adopt(self, dense: VectorQuantizedReRoPECache, layer_idx: int = 0) -> List[int]:
        """The sequences of a dense cache's layer (a prompt that one call prefilled), continued here; returns their ids.  Its counts belong
        to its codebook's entries and its queries to its rotary base: both have to be this cache's (a base it left to the model's
        configuration is not known here)."""
        assert self.rerope, "the dense cache holds ReRoPE keys"
        assert dense.window_length == self.window_length and tuple(dense.codebooks.shape) == tuple(self.codebooks.shape)
        if dense.rope_base is not None and dense.rope_base != self.rope_base:
            raise ValueError(f"the dense cache rotates with base {dense.rope_base}, this one with {self.rope_base}")
        other = dense.codebooks.to(self.device, torch.float32)
        if other.data_ptr() != self.codebooks.data_ptr() and not torch.equal(other, self.codebooks):
            raise ValueError("the dense cache counts codes of another codebook")
        st = dense.states[layer_idx]
        live, B = st["n"] - st["bd"], st["win_k3"].shape[0]
        if st["n"] > self.max_length:
            raise ValueError(f"a sequence of {st['n']} tokens exceeds max_length")
        if B > len(self._free_slots) or B * (-(-st["n"] // self.page_size) - st["bd"] // self.page_size) > len(self._free_pages):
            raise OutOfPages("the dense cache's sequences do not fit")
        sids = []
        try:
            for _ in range(B):
                sids.append(self.add_sequence())
            self._take_over(dense, st, [self._sequences[s] for s in sids], live)
        except BaseException:
            for s in sids:
                self.remove_sequence(s)
            raise
        return sids

    def _take_over(self, dense, st, seqs, live) -> None:
        B = len(seqs)
        for b, seq in enumerate(seqs):
            seq.n = seq.bd = st["bd"]
            seq.first = st["bd"] // self.page_size
            self.cnt[seq.slot].copy_(st["cnt"][b])
            self.vsum32[seq.slot].copy_(st["vsum32"][b])
            self.vsum[seq.slot].copy_(st["vsum32"][b])
        rows = lambda name: dense._window(st, name).transpose(1, 2).flatten(0, 1).to(self.dtype)
        lens = self._reserve(seqs, [live] * B) if live else [st["n"]] * B
        if live:
            meta = self._upload([live * i for i in range(B + 1)] + lens + [s.slot for s in seqs])
            api.paged_append(rows("win_k3"), rows("win_v"), self.pages, self.block_table.index_select(0, meta[2 * B + 1:]), meta[: B + 1],
                             meta[B + 1: 2 * B + 1], base=self.rope_base, n_pos=max(self.max_length, self.window_length + 2))
        for seq in seqs:
            seq.n = st["n"]

    def to_dense(self, sid: int) -> VectorQuantizedReRoPECache:
        """One sequence as a dense cache of its own (layer 0), window rows read back from their pages; the sequence stays here too."""
        assert self.rerope, "the dense cache holds ReRoPE keys"
        seq = self._sequences[sid]
        if seq.n == 0:
            raise ValueError("an empty sequence")
        meta = self._upload([seq.bd, seq.n])
        kv = self.pages
        k1, v, k3 = api.paged_read([(kv.k1, kv.k1_scale), (kv.v, kv.v_scale), (kv.k3, kv.k3_scale)], self.block_table[seq.slot: seq.slot + 1],
                                   meta[:1], meta[1:], seq.n - seq.bd, self.dtype)
        dense = VectorQuantizedReRoPECache(self.window_length, self.codebooks, False, rope_base=self.rope_base)
        s = seq.slot
        dense.update_prefill(self.cnt[s: s + 1].clone(), self.vsum32[s: s + 1].clone(), k1, v, 0, seq.n, {"key_unrotated": k3})
        return dense
