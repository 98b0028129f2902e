"""The status word of a device, used by several streams from its first use on."""
import pytest
import torch

from vqtree_b200 import native

pytestmark = pytest.mark.gpu


def test_what_another_stream_reports_is_not_cleared_by_the_first_use(monkeypatch):
    from vqtree_b200 import api
    k = torch.randn(3, 1, 64, device="cuda")
    pages = api.PagedKV.allocate(1, 1, 16, 64, torch.float32, "cuda", raw_keys=False)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    nowhere, cu, lens = i32(-1)[None], i32(0, 3), i32(3)
    api.paged_append(k, k, pages, i32(0)[None], cu, lens, rotate=False)     # the kernel is loaded
    api.check_status()
    monkeypatch.setattr(api, "_STATUS", {})
    busy = torch.randn(8192, 8192, device="cuda")
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):                                # no allocation of the driver's in between
        torch.empty(1, dtype=torch.int32, device="cuda")
        busy = busy @ busy * 1e-4
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        for _ in range(5):
            busy = busy @ busy * 1e-4                         # the word's zero waits behind some 30 ms
        api.device_status_word("cuda")
    with torch.cuda.stream(b):
        api.paged_append(k, k, pages, nowhere, cu, lens, rotate=False)
    torch.cuda.synchronize()
    with pytest.raises(native.VqError):
        api.check_status()
