"""The PyTorch C++ extension over the C ABI (torch.ops.vqattn.*): loading, schemas, sizes - no GPU needed."""
import re
from pathlib import Path

import pytest
import torch

from vqtree_b200 import native, torch_ops


@pytest.fixture(scope="module")
def ops():
    return torch_ops.load()


def test_extension_loads_and_reports_the_header_version(ops):
    header = (Path(__file__).resolve().parents[1] / "include" / "vqattn.h").read_text()
    assert int(ops.abi_version()) == int(re.search(r"#define VQATTN_VERSION (\d+)", header).group(1))


def test_workspace_sizes_equal_the_c_abi(ops):
    lib = native.lib
    assert ops.assign_workspace_bytes(1, 32, 32768, 4, 256, 128) == lib.vqattn_assign_workspace_bytes(1, 32, 32768, 4, 256, 128)
    assert ops.aggregates_workspace_bytes(2, 8, 3, 1, 512) == lib.vqattn_aggregates_workspace_bytes(2, 8, 3, 1, 512)
    assert ops.decode_workspace_bytes(16, 32, 32, 128) == lib.vqattn_decode_workspace_bytes(16, 32, 32, 128)


def test_operators_are_registered_as_out_variants(ops):
    for name in ("assign_codes", "build_aggregates", "prefill", "decode", "cache_advance"):
        schema = str(getattr(torch.ops.vqattn, name).default._schema)
        assert "-> ()" in schema and "(a!)" in schema, schema       # writes into its arguments, returns nothing


def test_there_is_no_cpu_kernel(ops):
    q = torch.zeros(1, 1, 128, 64)
    with pytest.raises(NotImplementedError):
        ops.prefill(q, q, q, q, q, None, None, None, 128, 0.0, 0, q.clone(), None, None)
    with pytest.raises(NotImplementedError):
        ops.assign_codes(q, torch.zeros(1, 1, 128, 64), None, torch.zeros(1, 1, 128, 1, dtype=torch.uint8), None, None)


def test_paged_operators_are_registered_in_both_forms(ops):
    for name in ("paged_append", "paged_read", "paged_attention"):
        assert "-> ()" in str(getattr(torch.ops.vqattn, name).default._schema) and "(a!)" in str(getattr(torch.ops.vqattn, name).default._schema)
        assert "-> int" in str(getattr(torch.ops.vqattn, name + "_status").default._schema)


def test_paged_entry_points_refuse_host_tensors():
    from vqtree_b200 import api
    z = torch.zeros
    i32 = lambda *s: z(*s, dtype=torch.int32)
    pages = api.PagedKV.allocate(2, 1, 16, 64, torch.float32, "cpu")
    with pytest.raises(ValueError):
        api.paged_append(z(3, 1, 64), z(3, 1, 64), pages, i32(1, 1), i32(2), i32(1))
    with pytest.raises(ValueError):
        api.paged_read([(pages.k1, None)], i32(1, 1), i32(1), i32(1), 3)
    with pytest.raises(ValueError):
        api.paged_attention(z(3, 1, 64), z(3, 1, 64), pages, i32(1, 1), i32(2), i32(1), 128, 3)
    with pytest.raises(ValueError):
        api.paged_attention(z(3, 1, 64), z(3, 1, 64), pages, i32(1, 1), i32(2), i32(1), 128, 3, codebook=z(1, 128, 64))
    with pytest.raises(ValueError):
        api.paged_read([], i32(1, 1), i32(1), i32(1), 3)
    assert api.paged_append(z(0, 1, 64), z(0, 1, 64), pages, i32(1, 1), i32(2), i32(1)) == (None, None)
    assert api.paged_attention(z(0, 1, 64), z(0, 1, 64), pages, i32(1, 1), i32(2), i32(1), 128, 1).shape == (0, 1, 64)
