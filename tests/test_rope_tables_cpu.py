"""The cached cos / sin tables: what a capture fills belongs to its graph."""
import torch

from vqtree_b200 import api


def test_a_table_filled_under_capture_is_not_cached(monkeypatch):
    monkeypatch.setattr(api, "_ROPE_TABLES", {})
    monkeypatch.setattr(api, "_ROPE_REPLACED", [])
    dev = torch.device("cpu", 0)
    with monkeypatch.context() as m:
        m.setattr(api, "_capturing", lambda d: True)
        cos, sin = api.rope_tables(40, 64, dev)
        assert cos.shape == sin.shape == (40, 32) and not api._ROPE_TABLES
    first = api.rope_tables(40, 64, dev)
    assert torch.equal(first[0], cos) and api.rope_tables(17, 64, dev) is first
    with monkeypatch.context() as m:                          # neither is one that a capture lengthens
        m.setattr(api, "_capturing", lambda d: True)
        assert api.rope_tables(40, 64, dev) is first
        assert api.rope_tables(41, 64, dev)[0].shape[0] >= 41
    assert api.rope_tables(40, 64, dev) is first and not api._ROPE_REPLACED
