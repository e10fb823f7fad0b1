"""The attention and rotary entries replaced by host functions: what the compiled callers (csrc/torch_calls.cpp) and their autograd nodes hand over can
be looked at on the CPU, on CPU tensors, without a kernel."""
import contextlib
import ctypes as C

import numpy as np
import torch

from dagnet_amd import _ops
from dagnet_amd._capi import DagnetHipError

VP, I32, I64 = C.c_void_p, C.c_int32, C.c_int64


class Attn(C.Structure):                       # dagnet_attn
    _fields_ = [(n, VP) for n in ("q", "k", "v", "slopes", "q_pos", "k_pos")] + \
               [(n, I64) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head")] + \
               [(n, I32) for n in ("nq", "nk", "n_heads", "n_kv_heads", "head_dim", "axes", "dtype", "max_keys", "mean_keys")] + \
               [("scale", C.c_float), ("softcap", C.c_float)]


def floats_at(address, n):
    return np.ctypeslib.as_array(C.cast(address, C.POINTER(C.c_float)), (n,)).copy() if n else np.zeros(0, np.float32)


def ints_at(address, n):
    return np.ctypeslib.as_array(C.cast(address, C.POINTER(C.c_int32)), (n,)).copy() if n else np.zeros(0, np.int32)


def rows_at(address, rows, heads, width, row, head):
    """fp32 [rows, heads, width] from a base and its strides."""
    if not rows:
        return np.zeros((0, heads, width), np.float32)
    flat = floats_at(address, (rows - 1) * row + (heads - 1) * head + width)
    return np.lib.stride_tricks.as_strided(flat, (rows, heads, width), (4 * row, 4 * head, 4)).copy()


def _copy(a):
    return Attn.from_buffer_copy(bytes(a.contents))


@contextlib.contextmanager
def recorded(on_fwd=None, on_bwd=None, on_step=None, on_rotary=None):
    """-> the callers, bound to entries that call on_*(name -> argument) and return 0; the library's own entries are bound again afterwards."""
    m = _ops.calls()
    seen = []                                            # exceptions of the callbacks: ctypes cannot raise them through C

    def entry(res, types, names, then):
        def call(*args):
            try:
                return (then(dict(zip(names, args))) if then else 0) or 0
            except BaseException as e:                   # noqa: BLE001
                seen.append(e)
                return 0
        return C.CFUNCTYPE(res, *types)(call)
    A = C.POINTER(Attn)

    def with_args(f):
        return None if f is None else lambda d: f({**d, "a": _copy(d["a"])})
    keep = {
        "dagnet_last_error": C.CFUNCTYPE(VP)(lambda: None),
        "dagnet_op_attn_fwd_workspace": entry(I64, (A,), ("a",), None),
        "dagnet_op_attn_fwd": entry(I32, (A,) + (VP,) * 7, ("a", "row_lo", "row_hi", "out", "lse", "o32", "workspace", "stream"), with_args(on_fwd)),
        "dagnet_op_attn_bwd_workspace": entry(I64, (A,), ("a",), None),
        "dagnet_op_attn_bwd": entry(I32, (A,) + (VP,) * 5 + (I64, I64) + (VP,) * 8, ("a", "row_lo", "row_hi", "key_lo", "key_hi", "dout", "do_row", "do_head", "lse", "o",
                                    "workspace", "dq", "dk", "dv", "dslopes", "stream"), with_args(on_bwd)),
        "dagnet_op_attn_step_workspace": entry(I64, (A, I32, I32, I32), ("a", "scenes", "room", "max_rows"), None),
        "dagnet_op_attn_step": entry(I32, (A, VP, VP, I32, I32, I32, I64, I64, VP, VP, VP), ("a", "q_ptr", "k_len", "scenes", "room", "max_rows", "k_scene", "v_scene",
                                     "out", "workspace", "stream"), with_args(on_step)),
        "dagnet_op_rotary": entry(I32, (I64, I32, I32, I32, I32, VP, I64, I64, VP, I64, I64, VP, I32, I32, VP, VP, I32, I32, I32, VP, I64, I64, VP, I64, I64, VP),
                                  ("n", "hq", "hk", "head_dim", "dtype", "q", "q_row", "q_head", "k", "k_row", "k_head", "pos", "pos_type", "axes", "turns", "axis",
                                   "pairs", "interleaved", "inverse", "qo", "qo_row", "qo_head", "ko", "ko_row", "ko_head", "stream"), on_rotary),
    }
    m.bind({n: C.cast(f, VP).value for n, f in keep.items()}, DagnetHipError)
    try:
        yield m
    finally:
        lib = _ops._lib()
        m.bind({n: C.cast(getattr(lib, n), VP).value for n in keep}, DagnetHipError)
    if seen:
        raise seen[0]


def host_tables(layout):
    """A layout's tables as the callers take them, in host memory of their own."""
    t = layout._host().clone()
    return layout._addresses(t) + (t,)


def host_axes(axes):
    t = axes._host().clone()
    return axes._addresses(t) + (t,)
