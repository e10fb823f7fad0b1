"""CPU: calls that torch's tracing, forward-mode differentiation and function transforms would see wrongly are refused before an entry is called (recorders
stand for the entries, tests/attn_recorder.py); gradients that come lazily are read as what they stand for."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from dagnet_amd import _ops
from dagnet_amd._capi import DagnetHipError
from dagnet_amd.attention import RotaryAxes, SceneLayout
from tests.attn_recorder import host_axes, host_tables, recorded, rows_at

N, H, KV, D = 6, 2, 1, 4
NAMES = ("scene_attn", "scene_attn_step", "rotary", "rotary_in_place")


def _tensors(name):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    if name == "scene_attn":
        return [r(N, H, D), r(N, KV, D), r(N, KV, D), r(H), r(N, 2), r(N, 2)]
    if name == "scene_attn_step":
        return [r(N, H, D), r(1, 9, KV, D), r(1, 9, KV, D), r(H), r(N, 2), r(1, 9, 2)]
    return [r(N, H, D), r(N, KV, D), r(N, 2)]


LAY, AX, LEN = host_tables(SceneLayout([0, N])), host_axes(RotaryAxes(D, (1, 1))), torch.tensor([3], dtype=torch.int32)


def _call(m, name, t):
    if name == "scene_attn":
        return m.scene_attn(*t[:4], LAY, 0.5, 0.0, *t[4:])
    if name == "scene_attn_step":
        return m.scene_attn_step(*t[:3], LEN, LAY[4], N, *t[3:], 0.5, 0.0)
    return m.rotary(*t, AX, 2, False, name == "rotary_in_place")[0]


@pytest.fixture
def entries():
    called = []
    note = lambda d: called.append(1)  # noqa: E731
    with recorded(on_fwd=note, on_bwd=note, on_step=note, on_rotary=note) as m:
        yield m, called


@pytest.mark.parametrize("name", NAMES)
def test_plain_tensors_go_through(entries, name):
    m, called = entries
    _call(m, name, _tensors(name))
    _call(m, name, [torch.nn.Parameter(t, requires_grad=False) for t in _tensors(name)])
    with torch.no_grad():
        _call(m, name, [t.requires_grad_() for t in _tensors(name)])
    with torch.inference_mode():
        _call(m, name, _tensors(name))
    assert len(called) == 4


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_not_lost(entries, name):
    m, called = entries
    for i in range(len(_tensors(name))):
        for grad in (False, True):
            t = _tensors(name)
            if grad and name != "rotary_in_place":
                t[0].requires_grad_()
            with fwd.dual_level(), pytest.raises(DagnetHipError, match="forward-mode"):
                t[i] = fwd.make_dual(t[i], torch.ones_like(t[i]))
                _call(m, name, t)
    assert not called


@pytest.mark.parametrize("name", NAMES)
def test_traces_are_refused(entries, name):
    m, called = entries
    t = _tensors(name)
    with pytest.raises(Exception, match="cannot be traced"):
        torch.jit.trace(lambda *a: _call(m, name, a), tuple(t), check_trace=False)
    assert not torch._C._get_tracing_state()
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(DagnetHipError, match="cannot be traced"):
            make_fx(lambda *a: _call(m, name, a), tracing_mode=mode)(*t)
    with FakeTensorMode() as mode, pytest.raises(DagnetHipError, match="cannot be traced"):
        _call(m, name, [mode.from_tensor(x) for x in t])
    with pytest.raises(DagnetHipError, match="plain tensors"):
        _call(m, name, [mode.from_tensor(x) for x in t])
    assert not called


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_refused(entries, name):
    m, called = entries
    t = _tensors(name)
    with pytest.raises(DagnetHipError, match="plain tensors"):
        torch.vmap(lambda q: _call(m, name, [q] + t[1:]))(torch.stack([t[0], t[0]]))
    with pytest.raises(DagnetHipError, match="plain tensors"):
        torch.func.grad(lambda q: _call(m, name, [q] + t[1:]).sum())(t[0])
    with pytest.raises(DagnetHipError, match="forward-mode|plain tensors"):
        torch.func.jvp(lambda q: _call(m, name, [q] + t[1:]), (t[0],), (t[0],))
    with pytest.raises(DagnetHipError, match="plain tensors|cannot be traced"):
        torch.func.functionalize(lambda q: _call(m, name, [q] + t[1:]))(t[0])
    assert not called


@pytest.mark.parametrize("name", NAMES)
def test_lazily_negated_views_are_refused(entries, name):
    """The memory of conj().imag holds the other sign."""
    m, called = entries
    for i in range(len(_tensors(name))):
        t = _tensors(name)
        t[i] = torch._neg_view(t[i])
        assert t[i].is_neg()
        with pytest.raises(DagnetHipError, match="resolve_neg"):
            _call(m, name, t)
    assert not called


def test_tables_are_not_made_under_a_fake_mode(monkeypatch):
    """A fake upload would be kept, and its address handed to a kernel later."""
    monkeypatch.setattr(_ops, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for x in (SceneLayout([0, 4]), RotaryAxes(8, (2,))):
        with FakeTensorMode(), pytest.raises(DagnetHipError, match="cannot be traced"):
            x.tables(0)
        assert x._dev == {}


@pytest.mark.parametrize("kind", ["negated", "zero", "transposed", "expanded"])
def test_lazy_gradients_are_read_as_what_they_stand_for(kind):
    g = torch.Generator().manual_seed(1)
    x = torch.randn((N, H, D), generator=g)
    dout = {"negated": torch._neg_view(x), "zero": torch._efficientzerotensor((N, H, D)), "transposed": x.transpose(1, 2).contiguous().transpose(1, 2),
            "expanded": torch.tensor(2.0).expand(N, H, D)}[kind]
    want = {"negated": -x, "zero": torch.zeros(N, H, D), "transposed": x, "expanded": torch.full((N, H, D), 2.0)}[kind].numpy()
    got = []
    with recorded(on_bwd=lambda d: got.append(rows_at(d["dout"], N, H, D, d["do_row"], d["do_head"])),
                  on_rotary=lambda d: got.append(rows_at(d["q"], N, H, D, d["q_row"], d["q_head"])) if d["inverse"] else None) as m:
        for name in ("scene_attn", "rotary"):
            t = _tensors(name)
            t[0].requires_grad_()
            torch.autograd.grad(_call(m, name, t), t[0], dout)
    assert len(got) == 2 and all(np.array_equal(a, want) for a in got)


@pytest.mark.parametrize("name", ["scene_attn", "rotary"])
def test_gradients_with_tangents_and_batched_ones_are_refused(entries, name):
    m, called = entries
    t = _tensors(name)
    t[0].requires_grad_()
    out = _call(m, name, t)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(out, t[0], fwd.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
    with pytest.raises(RuntimeError, match="plain tensors"):
        torch.autograd.grad(out, t[0], torch.ones((2,) + out.shape), is_grads_batched=True)
    assert len(called) == 1
