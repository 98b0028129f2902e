"""More refusals of the paged entry points of the C ABI, before they touch a device: -3 a stride, -4 host tensors (everything else is right), -7 an
argument."""
import ctypes

import pytest
import torch

z = torch.zeros


def _i32(*s):
    return z(*s, dtype=torch.int32)


def _native():
    from vqtree_b200 import native
    return native


def _attend(dtype, q8=False, T=7, **kw):
    native = _native()
    pool = lambda: z(4, 2, 16, 64, dtype=torch.int8 if q8 else dtype)
    scale = lambda: z(4, 2, 16) if q8 else None
    t = dict(k1=pool(), k3=pool(), v=pool(), k1_scale=scale(), k3_scale=scale(), v_scale=scale(), table=_i32(3, 5), cu_q=_i32(4), lens=_i32(3),
             **{n: z(T, 4, 64, dtype=dtype) for n in ("q1", "q2", "out")}, codebook=None, cnt=None, vsum=None, snap_table=None)
    t.update(kw)
    a = native.VqPagedAttentionArgs()
    for name, x in t.items():
        native.desc(x, getattr(a.kv if hasattr(a.kv, name) else a, name))
    a.window, a.max_q = 128, T
    return native.lib.vqattn_paged_attention(ctypes.byref(a), None)


@pytest.mark.parametrize("dtype,q8", [(torch.float32, False), (torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("T", [1, 7, 200])
def test_attention_refuses_expanded_rows_in_every_form(dtype, q8, T):
    assert _attend(dtype, q8, T) == -4
    for name in ("q1", "q2", "out"):
        assert _attend(dtype, q8, T, **{name: z(T, 1, 64, dtype=dtype).expand(T, 4, 64)}) == -3
        assert _attend(dtype, q8, T, **{name: z(1, 4, 64, dtype=dtype).expand(T, 4, 64)}) == (-4 if T == 1 else -3)
    kind = torch.int8 if q8 else dtype
    for name in ("k1", "k3", "v"):
        assert _attend(dtype, q8, T, **{name: z(4, 1, 16, 64, dtype=kind).expand(4, 2, 16, 64)}) == -3
        assert _attend(dtype, q8, T, **{name: z(1, 2, 16, 64, dtype=kind).expand(4, 2, 16, 64)}) == -3
    # one page table for all sequences, one scale for all rows: only read, and by plain loads
    assert _attend(dtype, q8, T, table=_i32(1, 5).expand(3, 5)) == -4
    if q8:
        assert _attend(dtype, q8, T, v_scale=z(1).expand(4, 2, 16)) == -4


def _append(**kw):
    native = _native()
    i8, sc, q = (lambda: z(4, 2, 16, 64, dtype=torch.int8)), (lambda: z(4, 2, 16)), (lambda: z(7, 4, 64))
    t = dict(k1=i8(), k3=i8(), v_pool=i8(), k1_scale=sc(), k3_scale=sc(), v_scale=sc(), table=_i32(3, 5), cu_q=_i32(4), lens=_i32(3), k=z(7, 2, 64),
             v=z(7, 2, 64), q=q(), q1=q(), q2=q())
    t.update(kw)
    a = native.VqPagedAppendArgs()
    native.desc(t.pop("v_pool"), a.kv.v)
    for name, x in t.items():
        native.desc(x, getattr(a.kv if name != "v" and hasattr(a.kv, name) else a, name))
    return native.lib.vqattn_paged_append(ctypes.byref(a), None)


def test_append_refuses_two_outputs_in_one_place():
    assert _append() == -4
    s, q = z(4, 2, 16), z(7, 4, 64)
    for pair in (("k1", "k3"), ("k1", "v"), ("k3", "v")):
        assert _append(**{n + "_scale": s for n in pair}) == -7
    assert _append(q1=q, q2=q) == -7
    # what is read may be one tensor, and queries may be rotated in place
    assert _append(q=q, q1=q) == -4 and _append(q2=None) == -4
    x = z(7, 2, 64)
    assert _append(k=x, v=x) == -4
