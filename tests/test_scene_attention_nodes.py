"""CPU: what the autograd nodes hand to the entries when saved-tensor hooks (activation checkpointing, offloading) put other tensors in the place of
the saved ones, and what they refuse.  The entries are recorders (tests/attn_recorder.py); no kernel runs."""
import gc

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from dagnet_amd.attention import RotaryAxes, SceneLayout
from tests.attn_recorder import floats_at, host_axes, host_tables, ints_at, recorded, rows_at

N, H, KV, D = 9, 4, 2, 8


def _inputs():
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    wide = r(N, (H + 2 * KV) * D)                                     # q, k and v as parts of one product
    q, k, v = (t.unflatten(1, (-1, D)) for t in wide.split([H * D, KV * D, KV * D], 1))
    return [q.clone().requires_grad_(), k.requires_grad_(), v.requires_grad_(), r(H).requires_grad_()], r(N, 2)


def _read(d):
    a = d["a"]
    return {"q": rows_at(a.q, a.nq, a.n_heads, a.head_dim, a.q_row, a.q_head), "k": rows_at(a.k, a.nk, a.n_kv_heads, a.head_dim, a.k_row, a.k_head),
            "v": rows_at(a.v, a.nk, a.n_kv_heads, a.head_dim, a.v_row, a.v_head), "slopes": floats_at(a.slopes, a.n_heads),
            "q_pos": floats_at(a.q_pos, a.nq * a.axes), "k_pos": floats_at(a.k_pos, a.nk * a.axes), "row_lo": ints_at(d["row_lo"], a.nq),
            "row_hi": ints_at(d["row_hi"], a.nq), "scale": a.scale, "cap": a.softcap, "span": (a.max_keys, a.mean_keys)}


def _fill(d):
    """The forward entry writes something that the backward has to find again."""
    a = d["a"]
    import ctypes as C
    np.ctypeslib.as_array(C.cast(d["out"], C.POINTER(C.c_float)), (a.nq * a.n_heads * a.head_dim,))[:] = 0.25
    np.ctypeslib.as_array(C.cast(d["lse"], C.POINTER(C.c_float)), (a.nq * a.n_heads,))[:] = np.arange(a.nq * a.n_heads)
    return 0


def _expect(got, leaves, pos, layout):
    for n, t in zip(("q", "k", "v", "slopes"), leaves):
        assert np.array_equal(got[n], t.detach().numpy()), n
    assert np.array_equal(got["q_pos"], pos.numpy().ravel()) and np.array_equal(got["k_pos"], pos.numpy().ravel())
    lo, hi = layout.row_bounds()
    assert np.array_equal(got["row_lo"], lo) and np.array_equal(got["row_hi"], hi) and got["span"] == layout.span
    assert got["scale"] == np.float32(0.3) and got["cap"] == 5.0


class _Moved:
    """Hooks that keep what they pack as copies at other places, with other strides, and spoil what was saved once the forward has gone."""

    def __init__(self, form="dense"):
        self.spoil, self.out, self.form = [], [], form

    def pack(self, t):
        self.spoil.append(t)
        return t.detach().clone()

    def unpack(self, t):
        if self.form == "dense":
            t = t.clone()
        elif self.form == "strided":                                   # the same values, every second element of a row
            t = torch.stack([t, t], -1)[..., 0]
        else:                                                          # the same values, their signs in memory the other way round
            t = torch._neg_view(-t)
            assert t.is_neg()
        self.out.append(t)
        return t


@pytest.mark.parametrize("form", ["dense", "strided", "negated"])
def test_the_backward_reads_what_the_hooks_return(form):
    leaves, pos = _inputs()
    layout = SceneLayout([0, 4, N], causal=1)
    got, hooks = [], _Moved(form)

    def on_bwd(d):
        got.append(_read(d))
        assert np.array_equal(floats_at(d["lse"], N * H), np.arange(N * H)) and (floats_at(d["o"], N * H * D) == 0.25).all()
        inside = [range(t.untyped_storage().data_ptr(), t.untyped_storage().data_ptr() + t.untyped_storage().nbytes()) for t in hooks.out]
        if form == "dense":                                            # and not what was saved
            for n in ("q", "k", "v", "slopes", "q_pos", "k_pos"):
                assert any(getattr(d["a"], n) in r for r in inside), n
    with recorded(on_fwd=_fill, on_bwd=on_bwd) as m:
        want = [t.detach().clone() for t in leaves]
        with torch.autograd.graph.saved_tensors_hooks(hooks.pack, hooks.unpack):
            out = m.scene_attn(*leaves, host_tables(layout), 0.3, 5.0, pos, pos)
        where = pos.clone()
        with torch.no_grad():
            for t in hooks.spoil:
                t.detach().fill_(-7.0) if t is not out else None
        torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert len(got) == 1
    _expect(got[0], want, where, layout)


def test_checkpointed_calls_read_what_was_computed_again():
    """Non-reentrant checkpointing frees what the first forward made: the projections, not the leaves, are what the node saw."""
    leaves, pos = _inputs()
    layout = SceneLayout([0, 4, N], causal=1)
    bwd = []
    with recorded(on_fwd=_fill, on_bwd=lambda d: bwd.append(_read(d))) as m:
        def block(q, k, v, s):
            return m.scene_attn(q * 2.0, k * 3.0, v + 1.0, s * 0.5, host_tables(layout), 0.3, 5.0, pos, pos)
        out = checkpoint(block, *leaves, use_reentrant=False)
        junk = [torch.full((N * H * D,), 9.0) for _ in range(64)]      # takes the memory of what was freed
        torch.autograd.grad(out, leaves, torch.ones_like(out))
        del junk
    assert len(bwd) == 1
    q, k, v, s = (t.detach() for t in leaves)
    _expect(bwd[0], [q * 2.0, k * 3.0, v + 1.0, s * 0.5], pos, layout)


def test_saving_on_the_host_and_a_layout_that_nobody_keeps():
    leaves, pos = _inputs()
    layout = SceneLayout([0, 4, N], causal=1)
    bwd = []
    with recorded(on_fwd=_fill, on_bwd=lambda d: bwd.append(_read(d))) as m:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.numpy(force=True).copy(), torch.from_numpy):
            out = m.scene_attn(*leaves, host_tables(layout), 0.3, 5.0, pos, pos)
        gc.collect()
        junk = [torch.full((len(layout._host()),), -1, dtype=torch.int32) for _ in range(64)]      # takes the memory of tables that are gone
        torch.autograd.grad(out, leaves, torch.ones_like(out))
        del junk
    _expect(bwd[0], leaves, pos, layout)


@pytest.mark.parametrize("change,match", [(lambda t: t.double(), "another shape, type or device"), (lambda t: t.reshape(-1), "another shape, type or device"),
                                          (lambda t: t.to("meta"), "another shape, type or device")])
@pytest.mark.parametrize("which", range(8))
def test_hooks_that_return_something_else_are_refused(which, change, match):
    """Before the entry is called.  Flattening is no change for what is flat already."""
    leaves, pos = _inputs()
    called, n = [], []

    def unpack(t):
        n.append(t)
        return change(t) if len(n) - 1 == which else t
    layout = SceneLayout([0, 4, N])
    with recorded(on_fwd=_fill, on_bwd=lambda d: called.append(1)) as m:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), unpack):
            out = m.scene_attn(*leaves, host_tables(layout), 0.3, 5.0, pos, pos)
        flat = change(torch.zeros(2, 2)).shape == (4,) and which in (3, 6)
        if flat:
            torch.autograd.grad(out, leaves, torch.ones_like(out))
        else:
            with pytest.raises(RuntimeError, match=match):
                torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert len(called) == flat


def test_rotary_reads_the_positions_that_the_hooks_return_and_its_own_tables():
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn((N, H, D), generator=g).requires_grad_(), torch.randn((N, KV, D), generator=g).requires_grad_()
    pos = torch.rand((N, 2), generator=g)
    want = pos.clone()
    axes = RotaryAxes(D, (2, 1))
    calls = []

    def on_rotary(d):
        calls.append((d["inverse"], floats_at(d["pos"], N * 2), floats_at(d["turns"], 2 * 3).view(np.float64), ints_at(d["axis"], 3)))
    with recorded(on_rotary=on_rotary) as m:
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.numpy(force=True).copy(), torch.from_numpy):
            a, b = m.rotary(q, k, pos, host_axes(axes), axes.n_pairs, False, False)
        gc.collect()
        junk = [torch.full((36,), 255, dtype=torch.uint8) for _ in range(64)]         # takes the memory of tables that are gone
        pos.fill_(-7.0)
        torch.autograd.grad((a, b), (q, k), (torch.ones_like(a), torch.ones_like(b)))
        del junk
    assert [c[0] for c in calls] == [0, 1]
    for _, p, turns, axis in calls:
        assert np.array_equal(p, want.numpy().ravel()) and np.array_equal(turns * 2 * np.pi, axes.freq) and axis.tolist() == axes.axis.tolist()


def test_rotary_refuses_other_positions_than_it_saved():
    q = torch.zeros(N, H, D, requires_grad=True)
    axes, calls = RotaryAxes(D, (2, 1)), []
    with recorded(on_rotary=lambda d: calls.append(1)) as m:
        for change in (lambda t: t[:3], lambda t: t.to(torch.int64)):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                a, _ = m.rotary(q, None, torch.zeros(N, 2), host_axes(axes), axes.n_pairs, False, False)
            with pytest.raises(RuntimeError, match="another shape, type or device"):
                torch.autograd.grad(a.sum(), q)
    assert len(calls) == 2
