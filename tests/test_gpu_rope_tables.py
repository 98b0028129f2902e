"""The cached cos / sin tables on several streams and under capture."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def api(monkeypatch):
    from vqtree_b200 import api as _api
    monkeypatch.setattr(_api, "_ROPE_TABLES", {})
    monkeypatch.setattr(_api, "_ROPE_REPLACED", [])
    return _api


def _append(api, n=300):
    """Keys of zeros and ones rotated into pages: the pages then hold the tables' entries."""
    k = torch.zeros(n, 1, 64, device="cuda")
    k[:, :, :32] = 1
    pages = api.PagedKV.allocate(5, 1, 64, 64, torch.float32, "cuda", raw_keys=False)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, cu, lens = torch.arange(5, dtype=torch.int32, device="cuda")[None], i32(0, n), i32(n)
    return pages, lambda: api.paged_append(k, k, pages, table, cu, lens, n_pos=1 << 17)


def _right(pages, n=300):
    """Angles of 64 bits, each table entry rounded once."""
    inv = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device="cuda") / 64)
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    want = torch.cat((ang.cos(), ang.sin()), 1)
    return (pages.k1[:, 0].flatten(0, 1)[:n] - want).abs().max().item() <= 2.0 ** -24


def test_a_second_stream_may_read_a_table_that_the_first_has_just_filled(api):
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    (p1, first), (p2, second) = _append(api), _append(api)
    busy = torch.randn(8192, 8192, device="cuda")
    for stream, call in ((a, first), (b, second)):            # kernels are loaded, memory is there
        with torch.cuda.stream(stream):
            call()
            busy @ busy
    torch.cuda.synchronize()
    api._ROPE_TABLES.clear()
    for p in (p1, p2):
        p.k1.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        for _ in range(5):
            busy = busy @ busy * 1e-4                         # the table waits behind some 30 ms
        first()
    with torch.cuda.stream(b):
        second()
    torch.cuda.synchronize()
    assert _right(p1) and _right(p2)


def test_a_first_use_under_capture_leaves_eager_calls_right_and_replays_right(api):
    (p1, captured), (p2, eager) = _append(api), _append(api)
    api.device_status_word("cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured()
    eager()
    assert _right(p2)
    graph.replay()
    assert _right(p1)
    p1.k1.zero_()
    torch.empty(1 << 26, device="cuda").fill_(float("nan"))
    graph.replay()
    assert _right(p1)
    api.check_status()
