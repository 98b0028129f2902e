"""Host logic of the paged cache (pages, snapshots, lengths) on the plain CPU forms of its operators."""
import pytest
import torch

from tests import fake_paged
from tests.paged_scenarios import serve, whole_sequences
from vqtree_b200.attn_vq import VectorQuantizedReRoPECache
from vqtree_b200.paged_cache import OutOfPages, PagedVectorQuantizedCache

W, D, M, K = 128, 64, 1, 128


@pytest.mark.parametrize("rerope", [True, False])
def test_chunks_of_every_size_equal_the_whole_prefill(rerope):
    cb, cases, want = whole_sequences((330, 150), 2, 1, D, M, K, W, torch.float32, rerope)
    # a prompt in pieces that span a boundary and two, single tokens next to them, a call that brings a sequence nothing
    schedule = [{0: 20}, {0: 110, 1: 140}, {1: 1, 0: 127}, {0: 1, 1: 1}, {0: 0, 1: 3}, {0: 70, 1: 5}, {0: 2}]
    with fake_paged.installed():
        got, cache, sids = serve(cases, cb, schedule, W, torch.float32, "cpu", rerope=rerope, page_size=16)
    for i in got:
        assert (got[i] - want[i][: got[i].shape[0]]).abs().max() <= 1e-4
    assert cache.length(sids[0]) == 330
    # live rows only: from the boundary of the last query on
    for i, n in ((0, 330), (1, 150)):
        bd = max(0, (n - 1 - W) // 128 * 128)
        seq = cache._sequences[sids[i]]
        assert seq.bd == bd and seq.first == bd // 16 and len(seq.pages) == -(-n // 16) - bd // 16
    held = sum(len(cache._sequences[s].pages) for s in sids.values())
    assert cache.free_pages == 64 - held
    used = [p for s in sids.values() for p in cache._sequences[s].pages]
    assert len(set(used) | set(cache._free_pages)) == 64
    for s in sids.values():
        cache.remove_sequence(s)
    assert cache.free_pages == 64


def test_slots_and_pages_are_reused_without_leaving_traces():
    cb, cases, want = whole_sequences((300, 40), 1, 1, D, M, K, W, torch.float32)
    with fake_paged.installed():
        cache = PagedVectorQuantizedCache(W, cb, 40, 1, page_size=16, dtype=torch.float32, device="cpu", max_length=512)
        for i, n in ((0, 300), (1, 40), (0, 300)):
            s = cache.add_sequence()
            with pytest.raises(OutOfPages):
                cache.add_sequence()
            got = cache.attend([s], [n], *cases[i]).view(n, 1, D)
            assert (got - want[i]).abs().max() <= 1e-4
            cache.remove_sequence(s)


def test_a_call_that_does_not_fit_changes_nothing():
    cb, cases, want = whole_sequences((300,), 1, 1, D, M, K, W, torch.float32)
    q, k, v = cases[0]
    with fake_paged.installed():
        cache = PagedVectorQuantizedCache(W, cb, 9, 2, page_size=32, dtype=torch.float32, device="cpu", max_length=512, spare_snapshots=0)
        s = cache.add_sequence()
        with pytest.raises(OutOfPages):
            cache.attend([s], [300], q, k, v)               # ten pages
        with pytest.raises(OutOfPages):                     # nine pages, but two boundaries and no spare snapshot
            cache.attend([s], [256 + 1], q[:257], k[:257], v[:257])
        assert cache.length(s) == 0 and cache.free_pages == 9
        got = cache.attend([s], [200], q[:200], k[:200], v[:200])
        with pytest.raises(OutOfPages):                     # two boundaries in one call, and no spare snapshot
            cache.attend([s], [57], q[200:257], k[200:257], v[200:257])
        got = torch.cat((got, cache.attend([s], [56], q[200:256], k[200:256], v[200:256]), cache.attend([s], [1], q[256:257], k[256:257], v[256:257])))
        assert (got.view(257, 1, D) - want[0][:257]).abs().max() <= 1e-4
        with pytest.raises(ValueError):
            cache.attend([s, s], [1, 1], q[:2], k[:2], v[:2])
        with pytest.raises(ValueError):
            cache.attend([s], [2], q[:1], k[:1], v[:1])
        with pytest.raises(ValueError):
            cache.attend([s], [1], q[:1].half(), k[:1].half(), v[:1].half())
        with pytest.raises(ValueError):
            cache.attend([s], [400], torch.zeros(400, 1, D), torch.zeros(400, 1, D), torch.zeros(400, 1, D))    # max_length
        assert cache.attend([s], [0], q[:0], k[:0], v[:0]).shape == (0, D) and cache.length(s) == 257


def test_to_dense_and_back():
    cb, cases, want = whole_sequences((290,), 2, 1, D, M, K, W, torch.float32)
    q, k, v = cases[0]
    with fake_paged.installed():
        cache = PagedVectorQuantizedCache(W, cb, 40, 3, page_size=16, dtype=torch.float32, device="cpu", max_length=512)
        s = cache.add_sequence()
        cache.attend([s], [280], q[:280], k[:280], v[:280])
        dense = cache.to_dense(s)
        assert isinstance(dense, VectorQuantizedReRoPECache) and dense.get_seq_length(0) == 280
        t, = cache.adopt(dense)
        for x in (s, t):
            got = cache.attend([x], [10], q[280:], k[280:], v[280:]).view(10, 2, D)
            assert (got - want[0][280:]).abs().max() <= 1e-4
