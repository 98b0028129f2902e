"""Paged calls whose tensors lie on two devices, and a cache whose device is not the current one."""
import pytest
import torch

from vqtree_b200 import native

pytestmark = pytest.mark.gpu

two = pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two devices")


@pytest.fixture(scope="module")
def api():
    from vqtree_b200 import api as _api
    return _api


@two
def test_workspaces_and_tables_of_another_device_are_refused(api):
    from tests.paged_cases import Case
    from vqtree_b200 import torch_ops
    c = Case(5, (600,), (700,), 1, 4, 64, 64, 128, 128, torch.bfloat16, True, True)
    need = api.paged_attention_workspace_bytes(1, 600, 4, 64, 1, 128, 600, torch.int8, torch.bfloat16)
    with pytest.raises(native.VqError) as e:
        c.attend(api, workspace=torch.empty(need, dtype=torch.uint8, device="cuda:1"))
    assert e.value.status == -4
    ops, k = torch_ops.load(), torch.zeros(3, 1, 64, device="cuda:0")
    p = api.PagedKV.allocate(1, 1, 16, 64, torch.float32, "cuda:0", raw_keys=False)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda:0")
    cos, sin = api.rope_tables(64, 64, "cuda:1")
    with pytest.raises(RuntimeError, match="status -4"):
        ops.paged_append(k, k, *p, i32(0)[None], i32(0, 3), i32(3), None, None, None, cos, sin, 0, None)


def _serve(cache, other):
    s = cache.add_sequence()
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(150, 1, 64, generator=g).cuda(0) for _ in range(3))
    got = []
    for a, b, dev in ((0, 140, 0), (140, 149, other), (149, 150, 0)):
        with torch.cuda.device(dev):
            got.append(cache.attend([s], [b - a], q[a:b], k[a:b], v[a:b]))
    cache.remove_sequence(s)
    return torch.cat(got)


def test_a_cache_belongs_to_the_device_that_was_current_when_it_was_made(api):
    from vqtree_b200.paged_cache import PagedVectorQuantizedCache
    cb = torch.randn(1, 1, 128, 64, generator=torch.Generator().manual_seed(4))
    cache = PagedVectorQuantizedCache(128, cb, 16, 2, page_size=16, dtype=torch.float32, max_length=256)
    assert cache.device == cache.codebooks.device == cache.pages.k1.device == torch.device("cuda", 0)
    other = 1 if torch.cuda.device_count() > 1 else 0
    assert torch.equal(_serve(cache, other), _serve(cache, 0))
    api.check_status("cuda:0")
