"""CPU: the layouts' row and key bounds against a row-by-row reading of their definition, and what the entry points refuse."""
import copy
import ctypes as C
import pickle
import random

import numpy as np
import pytest
import torch

from dagnet_amd import _capi, _ops, attention
from dagnet_amd._capi import DagnetHipError
from dagnet_amd.attention import RotaryAxes, SceneLayout, rotary, scene_attention, scene_attention_step
from tests import scene_attn_ref as ref


@pytest.mark.parametrize("q,k,causal,prefix", [
    ([0, 1], None, 0, 0), ([0, 3, 3, 10], None, 0, 0), ([0, 12, 20], None, 1, 0), ([0, 12, 20], None, [3, 4], [6, 0]), ([0, 12, 21], None, 5, 7),
    ([0, 4, 6], [0, 9, 20], 1, 0), ([0, 9, 20], [0, 4, 6], 1, 0), ([0, 9, 20], [0, 4, 6], 4, 2), ([0, 5, 5], [0, 0, 7], 0, 0), ([0, 0], [0, 4], 0, 0),
    ([0, 7, 9], [0, 30, 31], 0, 0), ([0, 5], None, 9, 100)])
def test_row_and_key_bounds(q, k, causal, prefix):
    lay = SceneLayout(q, k, causal=causal, prefix=prefix)
    seen = ref.seen_matrix(q, k, causal, prefix).numpy()
    lo, hi = lay.row_bounds()
    j = np.arange(lay.nk)[None, :]
    assert np.array_equal((j >= lo[:, None]) & (j < hi[:, None]), seen)
    assert np.all(np.diff(lo) >= 0) and np.all(np.diff(hi) >= 0)
    n, m = lay.nq, lay.nk
    klo, khi = lay._tab[2 * n:2 * n + m], lay._tab[2 * n + m:2 * n + 2 * m]
    assert np.all(np.diff(klo) >= 0) and np.all(np.diff(khi) >= 0)
    for c in range(m):
        rows = np.flatnonzero(seen[:, c])
        assert rows.size == 0 or (klo[c] <= rows[0] and rows[-1] < khi[c])
    assert np.all(klo >= 0) and np.all(khi <= n)


def test_seq_start_end_names_the_same_layout():
    a, b = SceneLayout([0, 4, 9]), SceneLayout(torch.tensor([[0, 4], [4, 9]]))
    assert np.array_equal(a._tab, b._tab) and a.S == b.S == 2 and a.max_rows == 5


@pytest.mark.parametrize("kw,match", [
    (dict(ptr=[1, 4]), "row pointers"), (dict(ptr=[0, 4, 3]), "row pointers"), (dict(ptr=[0]), "row pointers"), (dict(ptr=[0.0, 4.0]), "whole numbers"),
    (dict(ptr=[0, 4], k_ptr=[0, 4, 8]), "scenes"), (dict(ptr=[0, 4], causal=-1), "negative"), (dict(ptr=[0, 4], causal=[1, 2]), "per scene"),
    (dict(ptr=[0, 4], prefix=2), "needs causal"), (dict(ptr=[0, 4], causal=1.5), "whole number"), (dict(ptr=[[0, 4], [5, 9]]), "gaps"),
    (dict(ptr=[0, 2 ** 31]), "too many"), (dict(ptr=[0, 4], device="cpu"), "no CPU fallback")])
def test_layouts_refuse(kw, match):
    with pytest.raises(DagnetHipError, match=match):
        SceneLayout(**kw)


def _args(**kw):
    a = dict(q=torch.zeros(8, 4, 16), k=torch.zeros(8, 2, 16), v=torch.zeros(8, 2, 16), layout=SceneLayout([0, 8]))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(), "no CPU path"), (dict(layout=[0, 8]), "SceneLayout"), (dict(q=torch.zeros(8, 64)), "q must be"), (dict(q=torch.zeros(7, 4, 16)), "8 rows"),
    (dict(k=torch.zeros(8, 3, 16), v=torch.zeros(8, 3, 16)), "no multiple"), (dict(k=torch.zeros(8, 2, 8), v=torch.zeros(8, 2, 8)), "head_dim"),
    (dict(v=torch.zeros(8, 2, 8)), "one shape"), (dict(q=torch.zeros(8, 4, 129)), "1 .. 128"), (dict(q=torch.zeros(8, 4, 16).half()), "fp32 or all bf16"),
    (dict(k=torch.zeros(8, 2, 16).bfloat16()), "fp32 or all bf16"), (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"),
    (dict(scale=float("nan")), "scale"), (dict(pos=torch.zeros(8, 2)), "slopes"), (dict(slopes=torch.zeros(2), pos=torch.zeros(8, 2)), "slopes must be"),
    (dict(slopes=torch.zeros(4).double(), pos=torch.zeros(8, 2)), "slopes must be"), (dict(slopes=torch.zeros(4), pos=torch.zeros(8, 4)), "pos must be"),
    (dict(slopes=torch.zeros(4), pos=torch.zeros(8, 2).double()), "pos must be"), (dict(slopes=torch.zeros(4), pos=torch.zeros(8)), "pos must be"),
    (dict(slopes=torch.zeros(4), pos=torch.zeros(8, 2), k_pos=torch.zeros(8, 1)), "axes"), (dict(slopes=torch.zeros(4), k_pos=torch.zeros(8, 1)), "without pos"),
    (dict(slopes=torch.zeros(4), pos=torch.zeros(8, 2, requires_grad=True)), "no gradient"),
    (dict(layout=SceneLayout([0, 8], [0, 8]), slopes=torch.zeros(4), pos=torch.zeros(8, 2)), "k_pos is missing")])
def test_scene_attention_refuses(kw, match):
    with pytest.raises(DagnetHipError, match=match):
        scene_attention(**_args(**kw))


def _step(**kw):
    a = dict(q=torch.zeros(8, 4, 16), k_cache=torch.zeros(2, 30, 2, 16), v_cache=torch.zeros(2, 30, 2, 16), k_len=torch.zeros(2, dtype=torch.int32),
             layout=SceneLayout([0, 3, 8]))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(), "no CPU path"), (dict(layout=SceneLayout([0, 3, 8], causal=1)), "new rows only"), (dict(layout=SceneLayout([0, 3, 8], [0, 3, 8])), "new rows only"),
    (dict(k_len=torch.zeros(2, dtype=torch.int64)), "int32"), (dict(k_len=torch.zeros(3, dtype=torch.int32)), "int32"), (dict(k_len=[1, 2]), "int32"),
    (dict(layout=SceneLayout([0, 8])), "2 scenes"), (dict(k_cache=torch.zeros(30, 2, 16)), "key heads"), (dict(v_cache=torch.zeros(2, 29, 2, 16)), "one shape"),
    (dict(q=torch.zeros(8, 4, 16, requires_grad=True)), "no gradient"), (dict(k_pos=torch.zeros(2, 30, 1)), "slopes"),
    (dict(slopes=torch.zeros(4)), "pos must be"), (dict(slopes=torch.zeros(4), pos=torch.zeros(8, 1), k_pos=torch.zeros(2, 29, 1)), "k_pos must be")])
def test_step_refuses(kw, match):
    with pytest.raises(DagnetHipError, match=match):
        scene_attention_step(**_step(**kw))


@pytest.mark.parametrize("args,kw,match", [
    ((16, (5, 4)), {}, "pairs"), ((16, ()), {}, "pairs"), ((16, (-1, 4)), {}, "pairs"), ((16, (0,)), {}, "pairs"), ((2000, (8,)), {}, "pairs"),
    ((16, (4,)), dict(theta=0.0), "theta"), ((16, (4,)), dict(theta=float("inf")), "theta")])
def test_rotary_axes_refuse(args, kw, match):
    with pytest.raises(DagnetHipError, match=match):
        RotaryAxes(*args, **kw)


def _rot(**kw):
    a = dict(q=torch.zeros(6, 4, 16), k=torch.zeros(6, 2, 16), pos=torch.zeros(6, 2), axes=RotaryAxes(16, (4, 4)))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(), "no CPU path"), (dict(axes=(4, 4)), "RotaryAxes"), (dict(q=torch.zeros(6, 64)), "q must be"), (dict(k=torch.zeros(5, 2, 16)), "k must be"),
    (dict(k=torch.zeros(6, 2, 16).bfloat16()), "both be fp32"), (dict(pos=torch.zeros(6, 3)), "pos must be"), (dict(pos=torch.zeros(6, 2).double()), "pos must be"),
    (dict(q=torch.zeros(6, 4, 16, requires_grad=True), inplace=True), "no gradient"), (dict(q=torch.zeros(1, 4, 16).expand(6, 4, 16), inplace=True), "of its own"),
    (dict(pos=torch.zeros(6, 2, requires_grad=True)), "no gradient")])
def test_rotary_refuses(kw, match):
    with pytest.raises(DagnetHipError, match=match):
        rotary(**_rot(**kw))


def test_rotary_frequencies():
    a = RotaryAxes(32, (4, 0, 8), theta=(100.0, 5.0, 10000.0))
    assert a.axis.tolist() == [0] * 4 + [2] * 8 and a.n_pairs == 12
    assert np.allclose(a.freq[:4], [100.0 ** (-i / 4) for i in range(4)], rtol=1e-15)
    t = a._host().numpy()
    assert np.allclose(t[:96].view(np.float64) * 2 * np.pi, a.freq, rtol=1e-15) and t[96:].view(np.int32).tolist() == a.axis.tolist()


class _Attn(C.Structure):                       # dagnet_attn
    _fields_ = [(n, C.c_void_p) for n in ("q", "k", "v", "slopes", "q_pos", "k_pos")] + \
               [(n, C.c_int64) for n in ("q_row", "q_head", "k_row", "k_head", "v_row", "v_head")] + \
               [(n, C.c_int32) for n in ("nq", "nk", "n_heads", "n_kv_heads", "head_dim", "axes", "dtype", "max_keys", "mean_keys")] + \
               [("scale", C.c_float), ("softcap", C.c_float)]


def test_the_callers_load_and_bind():
    m = _ops.calls()
    assert m is _ops.calls() and all(hasattr(m, n) for n in ("scene_attn", "scene_attn_step", "rotary"))


def test_missing_callers_fail_loudly(monkeypatch):
    monkeypatch.setattr(_ops, "_calls", None)
    monkeypatch.setattr(_ops.os.path, "exists", lambda p: not p.endswith("_dagnet_torch.so"))
    with pytest.raises(DagnetHipError, match="no fallback"):
        _ops.calls()


def test_c_entries_refuse_before_any_launch():
    """Status and message, no exception across the boundary; none of these reaches a kernel."""
    lib = _ops._lib()
    ok = dict(nq=4, nk=4, n_heads=2, n_kv_heads=1, head_dim=16, axes=0, dtype=0, scale=1.0, softcap=0.0, q=64, k=64, v=64)

    def rc(**kw):
        a = _Attn(**{**ok, **kw})
        return lib.dagnet_op_attn_fwd(C.byref(a), *[None] * 7)
    for kw, word in ((dict(head_dim=129), b"head_dim"), (dict(head_dim=0), b"head_dim"), (dict(n_heads=3, n_kv_heads=2), b"multiple"), (dict(dtype=2), b"dtype"),
                     (dict(axes=4), b"axes"), (dict(max_keys=-1), b"max_keys"), (dict(nq=-1), b"row counts"), (dict(softcap=float("nan")), b"softcap"), (dict(scale=float("inf")), b"scale"),
                     (dict(q=None), b"null q"), (dict(axes=2), b"positions"), (dict(), b"null argument")):
        assert rc(**kw) == -1 and word in lib.dagnet_last_error()
    assert lib.dagnet_op_attn_fwd(None, *[None] * 7) == -1
    assert rc(nq=0, q=None) == 0
    a = _Attn(**ok)
    assert lib.dagnet_op_attn_bwd(C.byref(a), *[None] * 5, 0, 0, *[None] * 3, 64, 64, None, None, None) == -1 and b"dk and dv" in lib.dagnet_last_error()
    assert lib.dagnet_op_attn_bwd(C.byref(a), *[None] * 5, 0, 0, *[None] * 3, 64, None, None, 64, None) == -1 and b"dslopes" in lib.dagnet_last_error()
    assert lib.dagnet_op_attn_bwd_workspace(C.byref(a)) >= 16
    assert lib.dagnet_op_attn_step(C.byref(a), None, None, 1, 8, 1, 0, 0, None, None, None) == -1
    assert lib.dagnet_op_attn_step_workspace(C.byref(a), 0, 8, 1) == 0
    r = [2, 1, 0, 16, 0, 64, 0, 0, None, 0, 0, 64, 0, 1, 64, 64, 4, 0, 0, 64, 0, 0, None, 0, 0, None]
    for i, v in ((3, 1), (4, 2), (12, 3), (16, 9), (16, 0), (1, 0), (5, None)):
        bad = list(r)
        bad[i] = v
        assert lib.dagnet_op_rotary(*bad) == -1
    assert lib.dagnet_op_rotary(0, *r[1:]) == 0
    with pytest.raises(DagnetHipError, match="null argument"):
        _capi._check(lib.dagnet_op_attn_fwd(C.byref(a), *[None] * 7))


@pytest.mark.parametrize("make", [lambda: SceneLayout([0, 3, 8], causal=1), lambda: RotaryAxes(16, (4, 4))])
def test_copies_do_not_take_another_objects_addresses(make):
    a = make()
    a._dev[0] = ((1, 2, 3), 0)                       # as if uploaded
    for b in (copy.deepcopy(a), copy.copy(a), pickle.loads(pickle.dumps(a))):
        assert b._dev == {} and np.array_equal(b._host().numpy(), a._host().numpy())
    assert a._dev


@pytest.mark.parametrize("kw", [dict(softcap=1e-20), dict(softcap=1e20), dict(scale=1e20), dict(softcap=1e-46)])
def test_scales_that_leave_fp32_are_refused(kw):
    with pytest.raises(DagnetHipError, match="1e-15 .. 1e15"):
        scene_attention(**_args(**kw))


def _views(kind):
    n, H, KV, D = 6, 4, 2, 16
    if kind == "rows":                               # columns of one product
        x = torch.zeros(n, H + 2 * KV, D)
        return x[:, :H], x[:, H:H + KV]
    if kind == "heads":                              # q, k and v side by side in every head
        x = torch.zeros(n, H, 3, D)
        return x[:, :, 0], x[:, :, 1]
    if kind == "behind":                             # heads first
        x = torch.zeros(H + KV, n, D).transpose(0, 1)
        return x[:, :H], x[:, H:]
    x = torch.zeros(n, H, D)
    return {"same": (x, x), "part": (x, x[:, 1:3]), "shifted": (x.view(-1)[:n * 2 * D].view(n, 2, D), x.view(-1)[D:D + n * 2 * D].view(n, 2, D)),
            "windows": (x.view(-1).as_strided((n, 4, D), (16, 16, 1)), None)}[kind]


@pytest.mark.parametrize("kind,match", [("rows", "no CPU path"), ("heads", "no CPU path"), ("behind", "no CPU path"), ("same", "overlap"), ("part", "overlap"),
                                        ("shifted", "overlap"), ("windows", "of its own")])
def test_in_place_rotary_refuses_elements_that_are_turned_twice(kind, match):
    q, k = _views(kind)
    with pytest.raises(DagnetHipError, match=match):
        rotary(**_rot(q=q, k=k), inplace=True)


def test_what_the_strides_show_is_what_is():
    """Against the sets of elements: views that are called apart share none."""
    r = random.Random(3)
    x = torch.zeros(400)
    apart = 0
    for _ in range(2000):
        v = []
        for _ in range(2):
            shape = (r.randint(1, 4), r.randint(1, 3), r.choice((2, 4)))
            v.append(torch.as_strided(x, shape, (r.choice((4, 8, 16, 24)), r.choice((4, 8, 48)), 1), r.randint(0, 40)))
        sets = [(t.storage_offset() + (torch.arange(t.shape[0])[:, None, None] * t.stride(0) + torch.arange(t.shape[1])[:, None] * t.stride(1)
                                       + torch.arange(t.shape[2]))).flatten().tolist() for t in v]
        if attention._apart(*v):
            apart += 1
            assert not set(sets[0]) & set(sets[1])
        for t, s in zip(v, sets):
            assert not attention._own_elements(t) or len(set(s)) == len(s)
    assert apart > 500


def test_launches_that_cannot_be_counted_are_refused():
    lib = _ops._lib()
    a = _Attn(nq=2 ** 30, nk=4, n_heads=8, n_kv_heads=8, head_dim=16, axes=0, dtype=0, scale=1.0, softcap=0.0, q=64, k=64, v=64)
    assert lib.dagnet_op_attn_fwd(C.byref(a), *[64] * 3, None, None, None, None) == -1 and b"too many rows" in lib.dagnet_last_error()
    a.nq, a.nk = 4, 2 ** 30
    assert lib.dagnet_op_attn_fwd(C.byref(a), *[64] * 3, None, None, None, None) == -1 and b"too many rows" in lib.dagnet_last_error()
    assert lib.dagnet_op_rotary(16 * 0xffffff + 1, 1, 0, 16, 0, 64, 16, 16, None, 0, 0, 64, 0, 1, 64, 64, 4, 0, 0, 64, 16, 16, None, 0, 0, None) == -1
    assert b"too many rows" in lib.dagnet_last_error()
