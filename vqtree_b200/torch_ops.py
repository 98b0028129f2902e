"""``torch.ops.vqattn.*``: the PyTorch C++ extension over the library's C ABI.

``csrc/torch_ext.cpp`` registers the entry points of ``include/vqattn.h`` with PyTorch's dispatcher (CUDA
backend only - a CPU tensor finds no kernel and raises), each as an out-variant that writes into tensors the
caller passes: a C++ device guard, PyTorch's current stream, ``TORCH_CHECK`` errors.  The same kernels as the
ctypes layer (``native.py`` / ``api.py``) run; this binding is for callers that want dispatcher operators
(C++ callers, ``torch.compile`` graphs, TorchScript-free export) instead of a ctypes stub.

    from vqtree_b200 import torch_ops
    ops = torch_ops.load()                     # torch.ops.vqattn
    ops.prefill(q1, q2, k1, k3, v, cb_act, cnt, vsum, window, 0.0, 0, out, None, None)

Operators (argument meaning as in ``include/vqattn.h``; trailing ``status_word`` is the optional device int32
that kernels raise on an expired bounded wait or a bad code):
    assign_codes(k, codebooks, bias?, codes!, workspace?, status_word?)
    build_aggregates(codes, v, K, cnt!, vsum!, state_cnt!?, state_vsum!?, state_blocks, workspace?, status_word?)
    prefill(q1, q2, k1, k3, v, codebook?, cnt?, vsum?, window, scale, impl, out!, lse2!?, status_word?)
    decode(q1, q2, k1_win, k3_win, v_win, codebook?, cnt?, vsum?, n_valid, n_bd, scale, workspace!, out!, status_word?)
    cache_advance(codes, v_new, K, cnt!, vsum_f32!, vsum_act!?, status_word?)
    paged_append(k, v, k1!, v_pages!, k3!?, k1_scale!?, v_scale!?, k3_scale!?, table, cu_q, lens, q?, q1!?, q2!?, cos_tab?, sin_tab?,
                 const_pos, status_word?)
    paged_read(pool0, scale0?, out0!, pool1?, scale1?, out1!?, pool2?, scale2?, out2!?, table, start, lens, status_word?)
    paged_attention(q1, q2, k1, v_pages, k3?, k1_scale?, v_scale?, k3_scale?, table, cu_q, lens, codebook?, cnt?, vsum?, snap_table?,
                    window, max_q, scale, out!, workspace!?, status_word?)
    paged_*_status(...): the same, returning the C status instead of raising; paged_*_new(...): that, and the outputs allocated
    abi_version(), assign_workspace_bytes(...), aggregates_workspace_bytes(...), decode_workspace_bytes(...),
    paged_attention_workspace_bytes(S, T, Hq, Hkv, D, window, max_q, pool dtype, activations' dtype)
"""
from __future__ import annotations

from pathlib import Path

import torch

from . import native  # loads libvqattn.so first and fails loudly when it is missing

LIB = Path(__file__).resolve().parent / "lib" / "libvqattn_torch.so"
_PAGED = ("paged_append", "paged_read", "paged_attention")
_MUTATING = ("assign_codes", "build_aggregates", "prefill", "decode", "cache_advance") + _PAGED
_loaded = False


def load():
    """Loads the extension (once) and returns ``torch.ops.vqattn``."""
    global _loaded
    if not _loaded:
        if not LIB.exists():
            raise ImportError(f"{LIB} is missing: run `python -m vqtree_b200.build` (g++ against the installed torch)")
        torch.ops.load_library(str(LIB))
        if int(torch.ops.vqattn.abi_version()) != int(native.lib.vqattn_version()):
            raise ImportError("libvqattn_torch.so was built against another libvqattn.so: rebuild both")
        # shape propagation for tracing: the operators return nothing and only write into their arguments
        for name in _MUTATING:
            torch.library.register_fake(f"vqattn::{name}")(_nothing)
        for name in _PAGED:
            torch.library.register_fake(f"vqattn::{name}_status")(_ok)
        torch.library.register_fake("vqattn::paged_append_new")(lambda k, v, k1, vp, k3, a, b, c, t, cu, ln, q, two, *rest: (
            q.new_empty(q.shape), q.new_empty(q.shape if two else (0,)), 0))
        torch.library.register_fake("vqattn::paged_read_new")(lambda pools, scales, table, start, lens, n, dtype, word: (
            [p.new_empty((table.shape[0], p.shape[1], n, p.shape[3]), dtype=dtype) for p in pools], 0))
        torch.library.register_fake("vqattn::paged_attention_new")(lambda q1, *rest: (q1.new_empty(q1.shape), 0))
        _loaded = True
    return torch.ops.vqattn


def _nothing(*args, **kwargs):
    return None


def _ok(*args, **kwargs):
    return 0


def paged_calls():
    """What ``api.paged_*`` calls, looked up once: paged_append_status, paged_attention_status and the three ``*_new`` forms (describing some
    fifteen tensors in C++ takes 1 us, from Python 30)."""
    global _calls
    if _calls is None:
        ops = load()
        _calls = tuple(getattr(ops, n).default for n in ("paged_append_status", "paged_attention_status", "paged_append_new", "paged_read_new",
                                                         "paged_attention_new"))
    return _calls


_calls = None
