"""CPU-side checks of the C ABI: the library loads, exports what the header declares, and its
argument validation answers with the documented status codes before touching a device."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


def _native():
    from vqtree_b200 import native
    return native


def test_library_exports_every_declared_symbol():
    native = _native()
    header = (ROOT / "include" / "vqattn.h").read_text()
    declared = set(re.findall(r"\b(vqattn_[a-z_0-9]+)\s*\(", header))
    assert declared, "no declarations found"
    assert declared == set(native.EXPORTS)
    for name in declared:
        assert hasattr(native.lib, name)
    assert native.lib.vqattn_version() == int(re.search(r"#define VQATTN_VERSION (\d+)", header).group(1))


def test_struct_layout_matches_header():
    native = _native()
    # VqTensorDesc: ptr(8) dtype(4) ndim(4) shape(5*8) stride(5*8) device(4) + tail padding
    assert ctypes.sizeof(native.VqTensorDesc) == 104
    assert native.VqTensorDesc.shape.offset == 16 and native.VqTensorDesc.stride.offset == 56
    assert native.VqPrefillArgs.window.offset == 10 * 104
    assert native.VqDecodeArgs.n_valid.offset == 9 * 104


def test_aggregates_workspace_size():
    lib = _native().lib
    # per (batch, kv head, block, codebook): 128 key indices + K + 1 starts, rounded up to 16 bytes
    assert lib.vqattn_aggregates_workspace_bytes(1, 32, 247, 4, 256) == 32 * 247 * 4 * 400
    assert lib.vqattn_aggregates_workspace_bytes(2, 8, 3, 1, 512) == 2 * 8 * 3 * 656
    assert lib.vqattn_aggregates_workspace_bytes(0, 8, 3, 1, 512) == 0 and lib.vqattn_aggregates_workspace_bytes(1, 1, 1, 1, -4) == 0


def test_status_strings():
    native = _native()
    assert native.lib.vqattn_status_string(0) == b"ok"
    for code in range(-9, 0):
        assert native.lib.vqattn_status_string(code) not in (b"ok", b"unknown status")
    assert native.lib.vqattn_status_string(-99) == b"unknown status"


def test_validation_rejects_bad_arguments_without_a_device():
    native = _native()
    lib, desc = native.lib, native.desc
    k = torch.zeros(1, 2, 128, 64)
    cb = torch.zeros(2, 1, 128, 64)
    codes = torch.zeros(1, 2, 128, 1, dtype=torch.uint8)
    # null pointer
    assert lib.vqattn_assign_codes(None, desc(cb), None, desc(codes), None) == -7
    # wrong rank
    assert lib.vqattn_assign_codes(desc(k[0]), desc(cb), None, desc(codes), None) == -1
    # non-contiguous innermost dimension
    assert lib.vqattn_assign_codes(desc(k.transpose(2, 3)), desc(cb), None, desc(codes), None) == -3
    # host tensors are not on the current device (or there is no device): device error, not a crash
    assert lib.vqattn_assign_codes(desc(k), desc(cb), None, desc(codes), None) == -4
    # RoPE: null input, missing tables, no output asked for, constant position outside the tables, odd head dim
    x = torch.zeros(1, 2, 16, 64)
    tab = torch.zeros(32, 32)
    tp = ctypes.c_void_p(tab.data_ptr())
    assert lib.vqattn_rope(None, None, tp, tp, 32, 0, desc(x), None, None, None) == -7
    assert lib.vqattn_rope(desc(x), None, None, tp, 32, 0, desc(x), None, None, None) == -7
    assert lib.vqattn_rope(desc(x), None, tp, tp, 32, 0, None, None, None, None) == -7
    assert lib.vqattn_rope(desc(x), None, tp, tp, 32, 40, None, desc(x), None, None) == -7
    assert lib.vqattn_rope(desc(torch.zeros(1, 2, 16, 36)), None, tp, tp, 32, 0, desc(torch.zeros(1, 2, 16, 36)), None, None, None) == -1
    assert lib.vqattn_prefill(None, None) == -7
    assert lib.vqattn_decode(None, None) == -7
    assert lib.vqattn_decode_workspace_bytes(16, 32, 32, 128) >= 16 * 32 * 130 * 4


def test_missing_library_fails_loudly(tmp_path, monkeypatch):
    native = _native()
    monkeypatch.setattr(native, "_LIB_PATH", tmp_path / "nope.so")
    with pytest.raises(ImportError, match="no CPU or PyTorch fallback"):
        native._load()


def test_api_refuses_cpu_tensors():
    from vqtree_b200 import api
    with pytest.raises(ValueError):
        api.assign_codes(torch.zeros(1, 1, 128, 64), torch.zeros(1, 1, 128, 64))


def test_paged_entry_points_refuse_bad_arguments_without_a_device():
    native = _native()
    lib, desc = native.lib, native.desc
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)

    def append(**kw):
        t = dict(k1=torch.zeros(4, 2, 16, 64), k3=torch.zeros(4, 2, 16, 64), v_pool=torch.zeros(4, 2, 16, 64), table=i32(3, 5), cu_q=i32(4), lens=i32(3),
                 k=torch.zeros(7, 2, 64), v=torch.zeros(7, 2, 64), q=None, q1=None, q2=None, k1_scale=None, v_scale=None, k3_scale=None)
        tab = torch.zeros(32, 32)
        extra = dict(cos=tab.data_ptr(), sin=tab.data_ptr(), n_pos=32, const_pos=0)
        t.update({k: v for k, v in kw.items() if k in t})
        extra.update({k: v for k, v in kw.items() if k in extra})
        a = native.VqPagedAppendArgs()
        for name in ("k1", "k3", "table", "cu_q", "lens", "k1_scale", "v_scale", "k3_scale"):
            desc(t[name], getattr(a.kv, name))
        desc(t["v_pool"], a.kv.v)
        for name in ("k", "v", "q", "q1", "q2"):
            desc(t[name], getattr(a, name))
        a.cos_tab, a.sin_tab, a.n_pos, a.const_pos = extra["cos"], extra["sin"], extra["n_pos"], extra["const_pos"]
        return lib.vqattn_paged_append(ctypes.byref(a), None)

    z = torch.zeros
    assert append() == -4                                           # host tensors
    pool = z(4, 2, 16, 64)
    assert append(k1=pool, k3=pool) == -7 and append(k1=pool, v_pool=pool) == -7 and append(k3=None) == -4
    assert append(k=None) == -7 and append(k1=None) == -7 and append(v_pool=None) == -7
    assert append(k=z(7, 2, 64, dtype=torch.int32)) == -2 and append(k=z(7, 2, 64, dtype=torch.bfloat16)) == -2
    assert append(v=z(7, 3, 64)) == -1 and append(v=z(6, 2, 64)) == -1 and append(k=z(7, 2)) == -1
    assert append(v_pool=z(4, 2, 32, 64)) == -1 and append(k3=z(5, 2, 16, 64)) == -1
    assert append(k1=z(4, 2, 24, 64), k3=z(4, 2, 24, 64), v_pool=z(4, 2, 24, 64)) == -8      # page size
    assert append(k1=z(4, 2, 16, 32), k3=z(4, 2, 16, 32), v_pool=z(4, 2, 16, 32), k=z(7, 2, 32), v=z(7, 2, 32)) == -8
    assert append(k1=z(4, 2, 64, 16).transpose(2, 3)) == -3
    assert append(cu_q=i32(3)) == -1 and append(cu_q=z(4)) == -2 and append(lens=i32(4)) == -1 and append(table=z(3, 5)) == -2
    assert append(sin=None) == -7 and append(n_pos=0) == -7
    q = dict(q=z(7, 4, 64), q1=z(7, 4, 64))
    assert append(**q) == -4 and append(q=q["q"]) == -7 and append(q=q["q"], q1=z(7, 2, 64)) == -1
    assert append(**q, q2=z(7, 4, 64), const_pos=32) == -7 and append(**q, q2=z(7, 4, 64), const_pos=31) == -4
    assert append(k=z(7, 2, 65)[:, :, 1:]) == -3                    # rows that do not start on 16 bytes
    i8 = lambda: z(4, 2, 16, 64, dtype=torch.int8)
    sc = lambda: z(4, 2, 16)
    assert append(k1=i8(), k3=i8(), v_pool=i8()) == -7              # scales missing
    assert append(k1=i8(), k3=i8(), v_pool=i8(), k1_scale=sc(), k3_scale=sc(), v_scale=z(4, 2, 8)) == -1
    assert append(k1=i8(), k3=i8(), v_pool=i8(), k1_scale=sc(), k3_scale=sc(), v_scale=sc()) == -4
    assert append(v_scale=sc()) == -7                               # scales of rows that have none
    assert append(k1=z(1, 2, 16, 64).expand(4, 2, 16, 64)) == -3 and append(**dict(q, q1=z(1, 4, 64).expand(7, 4, 64))) == -3   # written to

    def read(pool, out, scale=None, table=i32(3, 5), start=i32(3), lens=i32(3)):
        a = native.VqPagedReadArgs()
        desc(pool, a.pool[0]); desc(out, a.out[0]); desc(scale, a.scale[0])
        desc(table, a.table); desc(start, a.start); desc(lens, a.lens)
        return lib.vqattn_paged_read(ctypes.byref(a), None)

    assert read(z(4, 2, 16, 64), z(3, 2, 9, 64)) == -4
    assert read(None, z(3, 2, 9, 64)) == -7 and read(z(4, 2, 16, 64), None) != 0
    assert read(z(4, 2, 16, 64), z(3, 2, 9, 64, dtype=torch.float16)) == -2 and read(z(4, 2, 16, 64, dtype=torch.int32), z(3, 2, 9, 64)) == -2
    assert read(z(4, 2, 16, 64), z(2, 2, 9, 64)) == -1 and read(z(4, 2, 16, 64), z(3, 2, 64, 9).transpose(2, 3)) == -3
    assert read(i8(), z(3, 2, 9, 64)) == -7 and read(i8(), z(3, 2, 9, 64), sc()) == -4

    def attend(**kw):
        t = dict(k1=z(4, 2, 16, 64), k3=z(4, 2, 16, 64), v=z(4, 2, 16, 64), table=i32(3, 5), cu_q=i32(4), lens=i32(3), q1=z(7, 4, 64), q2=z(7, 4, 64),
                 out=z(7, 4, 64), codebook=z(2, 128, 64), cnt=z(5, 2, 128), vsum=z(5, 2, 128, 64), snap_table=i32(3, 2))
        s = dict(window=128, max_q=7)
        t.update({k: v for k, v in kw.items() if k in t})
        s.update({k: v for k, v in kw.items() if k in s})
        a = native.VqPagedAttentionArgs()
        for name in ("k1", "k3", "v", "table", "cu_q", "lens"):
            desc(t[name], getattr(a.kv, name))
        for name in ("q1", "q2", "out", "codebook", "cnt", "vsum", "snap_table"):
            desc(t[name], getattr(a, name))
        a.window, a.max_q = s["window"], s["max_q"]
        return lib.vqattn_paged_attention(ctypes.byref(a), None)

    assert lib.vqattn_paged_attention(None, None) == -7 and lib.vqattn_paged_append(None, None) == -7 and lib.vqattn_paged_read(None, None) == -7
    assert attend() == -4 and attend(codebook=None) == -4
    assert attend(out=z(7, 1, 64).expand(7, 4, 64)) == -3
    assert attend(window=100) == -7 and attend(window=0) == -7 and attend(max_q=0) == -7
    assert attend(q1=z(7, 3, 64), q2=z(7, 3, 64), out=z(7, 3, 64)) == -1      # 3 query heads over 2
    assert attend(q2=z(7, 4, 64, dtype=torch.float16)) == -2 and attend(out=None) == -7 and attend(out=z(8, 4, 64)) == -1
    assert attend(codebook=z(2, 100, 64), cnt=z(5, 2, 100), vsum=z(5, 2, 100, 64)) == -8
    assert attend(cnt=z(4, 2, 128)) == -1 and attend(cnt=None) == -7 and attend(snap_table=i32(2, 2)) == -1 and attend(snap_table=z(3, 2)) == -2
    assert attend(vsum=z(5, 2, 64, 128).transpose(2, 3)) == -3
    assert attend(q1=z(7, 258, 64), q2=z(7, 258, 64), out=z(7, 258, 64)) == -8   # more than 128 query heads per kv head


def test_paged_attention_workspace_size():
    ws = _native().lib.vqattn_paged_attention_workspace_bytes
    # six sequences, 2228 new tokens of 4 query heads per kv head: three pools of 6 * (8 + 3) + 17 blocks of 128 rows and factors
    assert ws(6, 2228, 32, 8, 128, 1024, 597, 7, 1) == 3 * (6 * 11 + 17) * 8 * 128 * (128 * 2 + 4)
    assert ws(6, 2228, 32, 8, 128, 1024, 597, 1, 1) == 0            # rows of 16 bits
    assert ws(6, 2228, 32, 8, 128, 1024, 597, 7, 0) == 0            # full precision
    assert ws(17, 2228, 32, 8, 128, 1024, 597, 7, 1) > 0
    assert ws(18, 2228, 32, 8, 128, 1024, 597, 7, 1) == 0           # fewer than four tiles per sequence
    assert ws(1, 4, 32, 8, 128, 1024, 4, 7, 1) == 0 and ws(0, 0, 0, 0, 0, 0, 0, 7, 1) == 0 and ws(-1, 9, 4, 4, 128, 128, 9, 7, 1) == 0
