"""Calls of the paged cache that fail or are refused: they leave the cache as it was.  On the plain CPU forms of its operators."""
import pytest
import torch

from tests import fake_paged
from tests.paged_scenarios import whole_sequences
from vqtree_b200 import api
from vqtree_b200.attn_vq import VectorQuantizedReRoPECache
from vqtree_b200.paged_cache import OutOfPages, PagedVectorQuantizedCache, _runs

W, D, M, K = 128, 64, 1, 128


@pytest.fixture(scope="module")
def long_pair():
    return whole_sequences((500, 50), 2, 1, D, M, K, W, torch.float32)


def _cache(cb, **kw):
    kw = dict(dict(num_pages=64, max_sequences=3, page_size=16, dtype=torch.float32, device="cpu", max_length=1024), **kw)
    return PagedVectorQuantizedCache(W, cb, kw.pop("num_pages"), kw.pop("max_sequences"), **kw)


def _fail_once(monkeypatch, name, nth):
    """The nth call of api.<name> raises, as one that finds no memory does; those after it work again."""
    real, calls = getattr(api, name), [0]

    def call(*args, **kw):
        calls[0] += 1
        if calls[0] == nth:
            raise RuntimeError("out of memory")
        return real(*args, **kw)
    monkeypatch.setattr(api, name, call)


# a call of 300 after 200 tokens folds three blocks, of which two stand at boundaries of their own
@pytest.mark.parametrize("name,nth", [("paged_append", 1), ("paged_read", 1), ("assign_codes", 1), ("cache_advance", 1), ("cache_advance", 2),
                                      ("paged_attention", 1)])
@pytest.mark.parametrize("retry", [(300,), (100, 200)])
def test_a_call_that_fails_half_way_is_undone(monkeypatch, long_pair, name, nth, retry):
    cb, cases, want = long_pair
    part = lambda i, a, b: [x[a:b] for x in cases[i]]
    both = lambda x, y: [torch.cat(p) for p in zip(x, y)]
    with fake_paged.installed():
        cache = _cache(cb)
        a, b = cache.add_sequence(), cache.add_sequence()
        cache.attend([a, b], [200, 30], *both(part(0, 0, 200), part(1, 0, 30)))
        free = cache.free_pages
        with monkeypatch.context() as m:
            _fail_once(m, name, nth)
            with pytest.raises(RuntimeError, match="out of memory"):
                cache.attend([b, a], [20, 300], *both(part(1, 30, 50), part(0, 200, 500)))
        assert (cache.length(a), cache.length(b), cache.free_pages) == (200, 30, free)
        at = 200
        for q in retry:
            got = cache.attend([a], [q], *part(0, at, at + q)).view(q, 2, D)
            assert (got - want[0][at: at + q]).abs().max() <= 1e-4
            at += q
        got = cache.attend([b], [20], *part(1, 30, 50)).view(20, 2, D)
        assert (got - want[1][30:]).abs().max() <= 1e-4
        for s in (a, b):
            cache.remove_sequence(s)
        assert cache.free_pages == 64


def test_pages_of_a_failed_call_do_not_count_against_another_sequence(monkeypatch):
    cb, cases, want = whole_sequences((100, 60), 1, 1, D, M, K, W, torch.float32)
    with fake_paged.installed():
        cache = _cache(cb, num_pages=7)
        a, b = cache.add_sequence(), cache.add_sequence()
        with monkeypatch.context() as m:
            _fail_once(m, "paged_attention", 1)
            with pytest.raises(RuntimeError):
                cache.attend([a], [100], *cases[0])          # seven pages
        assert cache.free_pages == 7
        got = cache.attend([a, b], [16, 60], *(torch.cat((x[:16], y)) for x, y in zip(*cases)))
        assert (got.view(76, 1, D) - torch.cat((want[0][:16], want[1]))).abs().max() <= 1e-4


@pytest.mark.parametrize("heads", [3, 258, 0])
def test_query_heads_that_attention_would_refuse_are_refused_before_anything_changes(heads):
    cb = torch.randn(2, M, K, D)
    with fake_paged.installed():
        cache = _cache(cb)
        s = cache.add_sequence()
        k = torch.randn(20, 2, D)
        with pytest.raises(ValueError, match="heads"):
            cache.attend([s], [20], torch.randn(20, heads, D), k, k)
        with pytest.raises(ValueError):
            cache.attend([s], [20], torch.randn(20, 4, D), k.half(), k.half())
        assert cache.length(s) == 0 and cache.free_pages == 64


def _dense(n, cb, batch=2, **kw):
    """A dense cache as a prefill of n tokens leaves it: rows of ones, counts of zeros."""
    bd = max(0, (n - W) // 128 * 128)
    H, rows = cb.shape[0], torch.ones(batch, cb.shape[0], n - bd, D)
    dense = VectorQuantizedReRoPECache(W, cb, **kw)
    dense.update_prefill(torch.zeros(batch, H, M * K), torch.zeros(batch, H, M * K, D), rows, rows, 0, n, {"key_unrotated": rows})
    return dense


def test_adopt_that_is_refused_or_fails_keeps_no_slot_and_no_page(monkeypatch):
    cb = torch.randn(1, M, K, D)
    with fake_paged.installed():
        cache = _cache(cb, max_length=256)
        with pytest.raises(ValueError, match="max_length"):
            cache.adopt(_dense(300, cb))
        with pytest.raises(OutOfPages):
            cache.adopt(_dense(200, cb, batch=4))
        with monkeypatch.context() as m:
            _fail_once(m, "paged_append", 1)
            with pytest.raises(RuntimeError):
                cache.adopt(_dense(200, cb))
        assert cache.free_pages == 64
        sids = cache.adopt(_dense(200, cb, batch=3))          # all three slots
        assert [cache.length(s) for s in sids] == [200] * 3 and cache.free_pages == 64 - 3 * 13


def test_adopt_refuses_another_codebook_and_another_rotary_base():
    cb = torch.randn(1, M, K, D)
    with fake_paged.installed():
        cache = _cache(cb, rope_base=5e5)
        with pytest.raises(ValueError, match="base"):
            cache.adopt(_dense(200, cb, rope_base=1e4))
        with pytest.raises(ValueError, match="codebook"):
            cache.adopt(_dense(200, cb + 1, rope_base=5e5))
        assert cache.free_pages == 64
        # an equal codebook elsewhere, one of fewer bits that stands for the same numbers, a base left to the model's configuration
        cache.adopt(_dense(150, cb.clone(), batch=1, rope_base=5e5))
        cache.adopt(_dense(150, cb, batch=1))
        half = _cache(cb.half().float())
        half.adopt(_dense(150, cb.half(), batch=1))


def test_a_failed_call_of_many_sequences_restores_each(monkeypatch):
    """Blocks leave in three of four slots, two of them neighbours; sums, counts and boundaries are those of before, bit for bit."""
    assert [(s.start, s.stop) for s in _runs({7, 1, 3, 2})] == [(1, 4), (7, 8)] and _runs(set()) == []
    cb = torch.randn(1, M, K, D)
    n = (250, 250, 10, 250)
    with fake_paged.installed():
        cache = _cache(cb, max_sequences=4, num_pages=128)
        sids = [cache.add_sequence() for _ in n]
        cache.attend(sids, n, *(torch.randn(sum(n), 1, D) for _ in range(3)))
        held = [t.clone() for t in (cache.cnt, cache.vsum32, cache.vsum)]
        marks = [(s.n, s.bd, s.first, list(s.pages)) for s in cache._sequences.values()]
        with monkeypatch.context() as m:
            _fail_once(m, "paged_attention", 1)
            with pytest.raises(RuntimeError):
                cache.attend(sids, [150] * 4, *(torch.randn(600, 1, D) for _ in range(3)))
        for t, old in zip((cache.cnt, cache.vsum32, cache.vsum), held):
            assert torch.equal(t[:4], old[:4])
        assert [(s.n, s.bd, s.first, list(s.pages)) for s in cache._sequences.values()] == marks
