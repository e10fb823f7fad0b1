"""CPU: C entries of the attention with counts and addresses that have to be refused on the host; none of these calls reaches a kernel."""
import ctypes as C

import pytest

from dagnet_amd import _ops
from tests.attn_recorder import Attn


def _attn(**kw):
    return Attn(**{**dict(nq=4, nk=4, n_heads=2, n_kv_heads=1, head_dim=16, axes=0, dtype=0, scale=1.0, softcap=0.0, q=64, k=64, v=64), **kw})


@pytest.mark.parametrize("n_heads,max_rows", [(2 ** 20, 2 ** 16), (2 ** 20, 2 ** 31 - 1), (1, 2 ** 31 - 1), (2, 2 ** 29)])
def test_a_step_of_more_packed_rows_than_can_be_counted(n_heads, max_rows):
    """2^20 heads of one key head times 2^16 rows are 2^32 blocks of 16: 0 in 32 bits, and a division by it."""
    lib, a = _ops._lib(), _attn(nq=1, n_heads=n_heads)
    assert lib.dagnet_op_attn_step_workspace(C.byref(a), 1, 8, max_rows) == 0
    assert lib.dagnet_op_attn_step(C.byref(a), 64, 64, 1, 8, max_rows, 16, 16, 64, None, None) == -1 and b"too many rows" in lib.dagnet_last_error()


def test_a_step_of_more_scenes_than_can_be_counted():
    """2^30 scenes by 2^23 key heads by 2^11 blocks are 2^64."""
    lib, a = _ops._lib(), _attn(nq=1, n_heads=2 ** 23, n_kv_heads=2 ** 23)
    assert lib.dagnet_op_attn_step_workspace(C.byref(a), 2 ** 30, 8, 2 ** 15) == 0
    assert lib.dagnet_op_attn_step(C.byref(a), 64, 64, 2 ** 30, 8, 2 ** 15, 16, 16, 64, None, None) == -1 and b"too many rows" in lib.dagnet_last_error()


def test_a_step_refuses_a_workspace_between_two_floats_of_four():
    lib, a = _ops._lib(), _attn()
    assert lib.dagnet_op_attn_step_workspace(C.byref(a), 1, 8192, 4) > 0
    for ws in (None, 8, 68):
        assert lib.dagnet_op_attn_step(C.byref(a), 64, 64, 1, 8192, 4, 16, 16, 64, ws, None) == -1 and b"workspace" in lib.dagnet_last_error()
