"""GPU: attention and rotary calls as programs around them make them - under activation checkpointing and saved-tensor hooks, on empty batches, with a
scale of nothing, split over many workgroups beside spoilt rows, straight from the C entries."""
import ctypes as C
import gc

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from dagnet_amd import _ops
from dagnet_amd.attention import RotaryAxes, SceneLayout, rotary, scene_attention, scene_attention_step
from tests import scene_attn_ref as ref
from tests.attn_recorder import Attn
from tests.test_gpu_scene_attention import BF16, DEV, F32, both, inputs, randn, step_inputs, step_want

pytestmark = pytest.mark.gpu


def _block(q, k, v, slopes, pos, w):
    """A layer's call: projections whose memory nobody else holds, tables that only this call has."""
    axes = RotaryAxes(q.shape[2], (4, 4))
    layout = SceneLayout([0, 37, 90], causal=3)
    a, b = rotary(q * w, k * w, pos * 2.0, axes)
    return scene_attention(a, b, v + w, layout, softcap=10.0, slopes=slopes * 0.5, pos=pos * 1.0)


class _Copies(torch.autograd.graph.saved_tensors_hooks):
    def __init__(self):
        super().__init__(lambda t: t.detach().clone(), lambda t: t.clone())


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("how", ["checkpoint", "on_host", "copies"])
def test_gradients_under_hooks_equal_the_direct_ones(how, dt):
    t = inputs(13, 90, 90, 4, 2, 16, dt, 2)
    w = torch.tensor(1.25, device=DEV, dtype=dt)
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v", "slopes")]
    args = (*leaves, t["pos"], w)
    want = torch.autograd.grad(_block(*args), leaves, t["dout"])
    if how == "checkpoint":
        out = checkpoint(_block, *args, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu() if how == "on_host" else _Copies():
            out = _block(*args)
    gc.collect()
    junk = [torch.full((n,), 3, dtype=torch.int32, device=DEV) for n in (64, 400, 1440, 2880, 5760) for _ in range(24)]     # takes what was freed
    got = torch.autograd.grad(out, leaves, t["dout"])
    del junk
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-50, 1e-40])
@pytest.mark.parametrize("rows,lens,room", [([1], [1], 1), ([3, 2], [37, 90], 100), ([10, 1, 4], [1001, 0, 700], 1111)])
def test_a_step_with_a_scale_of_nothing_gives_the_mean(rows, lens, room, scale, dt):
    """Scores are 0 (1e-50 is 0 in fp32, 1e-40 a denormal): all kept keys weigh the same, one split of the keys or several."""
    t = step_inputs(room, rows, lens, room, 4, 2, 24, dt, 0)
    got = scene_attention_step(t["q"], t["k"], t["v"], t["k_len"], SceneLayout(t["ptr"]), scale=scale)
    want, tol = step_want(t, lens, 0.0, scale)
    ref.close(got, want["out"], tol["out"], "step")


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("scale", [0.0, 1e-40])
@pytest.mark.parametrize("ptr,causal", [([0, 5, 70], 1), ([0, 1, 300], 0), ([0, 700], 1)])
def test_a_scale_of_nothing_forward_and_backward(ptr, causal, scale, cap, dt):
    t = inputs(3, ptr[-1], ptr[-1], 4, 2, 24, dt, 0)
    both(t, SceneLayout(ptr, causal=causal), ref.seen_matrix(ptr, None, causal), scale=scale, cap=cap)


@pytest.mark.parametrize("axes", [1, 2, 3])
@pytest.mark.parametrize("q_ptr,k_ptr", [([0, 0], [0, 30]), ([0, 30], [0, 0]), ([0, 0], [0, 0]), ([0, 0, 7], [0, 12, 12])])
def test_no_rows_or_no_keys_with_learned_slopes(q_ptr, k_ptr, axes):
    t = inputs(1, q_ptr[-1], k_ptr[-1], 2, 2, 16, F32, axes)
    out, grads = both(t, SceneLayout(q_ptr, k_ptr), torch.zeros((q_ptr[-1], k_ptr[-1]), dtype=torch.bool))
    assert (out == 0).all() and all((g == 0).all() for g in grads) and grads[3].shape == (2,)


def test_an_empty_batch_trains_with_the_default_positions():
    q, k = torch.zeros((0, 2, 16), device=DEV, requires_grad=True), torch.zeros((0, 1, 16), device=DEV, requires_grad=True)
    slopes = torch.full((2,), 0.5, device=DEV, requires_grad=True)
    got = torch.autograd.grad(scene_attention(q, k, k, SceneLayout([0, 0, 0]), slopes=slopes).sum(), (q, k, slopes))
    assert got[0].shape == q.shape and got[1].shape == k.shape and (got[2] == 0).all()


def _step_entry(t, ptr, lens, max_rows, out, dtype):
    """dagnet_op_attn_step itself: rows of q that no scene owns can be named there only."""
    lib = _ops._lib()
    S, room, KV, D = t["k"].shape
    H = t["q"].shape[1]
    a = Attn(q=t["q"].data_ptr(), k=t["k"].data_ptr(), v=t["v"].data_ptr(), q_row=H * D, q_head=D, k_row=KV * D, k_head=D, v_row=KV * D, v_head=D, nq=t["q"].shape[0],
             nk=0, n_heads=H, n_kv_heads=KV, head_dim=D, axes=0, dtype=dtype, scale=D ** -0.5, softcap=0.0)
    q_ptr, k_len = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (ptr, lens))
    ws = torch.full((max(1, lib.dagnet_op_attn_step_workspace(C.byref(a), S, room, max_rows)),), 1e3, device=DEV)
    rc = lib.dagnet_op_attn_step(C.byref(a), q_ptr.data_ptr(), k_len.data_ptr(), S, room, max_rows, room * KV * D, room * KV * D, out.data_ptr(), ws.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc, ws.numel()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("room", [90, 700, 5000])
def test_rows_of_a_step_that_no_scene_owns_stay_as_they_were(room, dt):
    """Rows before the first scene's and behind the last one's, with the keys in one split (90) and in several."""
    ptr, lens = [1, 4, 4, 6], [room - 3, 5, room]
    t = step_inputs(room, [9, 0, 0], lens, room, 4, 2, 32, dt, 0)
    out = torch.full((9, 4, 32), 7.0, device=DEV, dtype=dt)
    rc, ws = _step_entry(t, ptr, lens, 3, out, int(dt is BF16))
    assert rc == 0 and (ws > 1) == (room > 256)
    assert (out[:1] == 7.0).all() and (out[6:] == 7.0).all()
    t["ptr"] = [0, 3, 3, 5]
    t["q"] = t["q"][1:6]
    want, tol = step_want(t, lens, 0.0, 32 ** -0.5)
    ref.close(out[1:6], want["out"], tol["out"], "step")


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("names", [("k", "v"), ("q", "dout"), ("dout",), ("q", "k", "v", "dout")])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_spoilt_rows_of_another_scene_do_not_reach_split_sums(names, bad, dt):
    """Two scenes whose border lies inside a tile, large enough that a tile's keys and a tile's rows are split over workgroups; rows of the second one are
    spoilt next to the border and far from it.  The first scene's results are those of the formulas, the keys beside the border among them."""
    ptr, H, KV, D = [0, 700, 1500], 4, 2, 24
    layout = SceneLayout(ptr)
    t = inputs(17, 1500, 1500, H, KV, D, dt, 1)
    lib, a = _ops._lib(), Attn(nq=1500, nk=1500, n_heads=H, n_kv_heads=KV, head_dim=D, axes=1, dtype=int(dt is BF16), max_keys=layout.span[0], mean_keys=layout.span[1])
    more = lib.dagnet_op_attn_bwd_workspace(C.byref(a)) - 2 * 1500 * H
    assert more >= 2 * 1500 * H * D + 2 * 2 * 1500 * KV * D              # at least two parts of the keys and of the rows
    cut = {n: t[n][:700].clone() for n in ("q", "k", "v", "dout", "pos")}
    for n in names:
        for i in (700, 705, 763, 1400):
            t[n][i] = bad
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v", "slopes")]
    out = scene_attention(*leaves[:3], layout, softcap=8.0, slopes=t["slopes"], pos=t["pos"])
    grads = torch.autograd.grad(out, leaves, t["dout"])
    assert not all(torch.isfinite(x[700:]).all() for x in (out,) + grads[:3])
    want, tol = ref.attention(cut["q"], cut["k"], cut["v"], ref.seen_matrix([0, 700]), D ** -0.5, 8.0, t["slopes"], cut["pos"], cut["pos"], cut["dout"])
    for name, got in zip(("out", "dq", "dk", "dv"), (out,) + grads[:3]):
        ref.close(got[:700], want[name], tol[name], name)


def test_sums_of_the_slopes_gradient_keep_their_bits_between_key_parts():
    """One row over 1024 keys in eight parts, all scores 0: p = 2^-10, the values' mean is 0, so dslope = -2^-10 sum_j v_j d_j.  With v = +-255 and whole distances
    below 2^12 every fp32 sum of a lane's 16 pairs is exact (16 2^20 = 2^24); a part's 128 need 27 bits, and the parts cancel to fewer than 24."""
    g = torch.Generator().manual_seed(2)
    n = 1024
    d = torch.randint(2 ** 11, 2 ** 12, (n,), generator=g).double() // 2 * 2 + 1
    v = torch.where(torch.arange(n) < n // 2, 255.0, -255.0)
    q, k = torch.zeros((1, 1, 1), device=DEV), torch.ones((n, 1, 1), device=DEV)
    slopes = torch.zeros(1, device=DEV, requires_grad=True)
    out = scene_attention(q, k, v.view(n, 1, 1).to(DEV), SceneLayout([0, 1], [0, n]), slopes=slopes, pos=torch.zeros((1, 1), device=DEV),
                          k_pos=d.float().view(n, 1).to(DEV))
    assert float(out.detach()) == 0.0
    got, = torch.autograd.grad(out, slopes, torch.ones_like(out))
    want = -float((v.double() * d).sum()) / n
    assert abs(want * n) < 2 ** 24 and float(got) == want


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N", [700, 3000])
def test_a_gradient_of_nan_gives_nan(N, dt):
    """What a loss that overflowed sends back: every key is taken one by one then."""
    t = inputs(2, N, N, 4, 2, 32, dt, 0)
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v")]
    out = scene_attention(*leaves, SceneLayout([0, N], causal=1))
    grads = torch.autograd.grad(out, leaves, torch.full_like(out, float("nan")))
    assert torch.isfinite(out).all() and all(g.isnan().all() for g in grads)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("axes", [0, 2])
def test_a_step_without_keys_or_rows(axes, dt):
    """A cache without room, one whose scenes keep nothing yet, and a step that brings no rows."""
    kw = lambda t: dict(slopes=t["slopes"], pos=t["pos"], k_pos=t["k_pos"]) if axes else {}  # noqa: E731
    for lens, room in (([0, 0], 0), ([0, 0], 700)):
        t = step_inputs(1, [3, 2], lens, room, 4, 2, 24, dt, axes)
        got = scene_attention_step(t["q"], t["k"], t["v"], t["k_len"], SceneLayout(t["ptr"]), softcap=5.0, **kw(t))
        assert got.shape == (5, 4, 24) and (got == 0).all()
    t = step_inputs(1, [0, 0], [5, 9], 20, 4, 2, 24, dt, axes)
    assert scene_attention_step(t["q"], t["k"], t["v"], t["k_len"], SceneLayout(t["ptr"]), **kw(t)).shape == (0, 4, 24)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_keys_and_values_that_are_one_tensor_or_broadcast(dt):
    """k and v the same leaf (both gradients meet in it), and k with one head or one row spread over all (strides 0): the spread ones' gradients add up."""
    ptr = [0, 30, 75]
    t = inputs(6, 75, 75, 4, 2, 16, dt, 0)
    layout, seen = SceneLayout(ptr, causal=1), ref.seen_matrix(ptr, None, 1)
    want, tol = ref.attention(t["q"], t["k"], t["k"], seen, 0.25, 0.0, None, None, None, t["dout"])
    q, k = t["q"].requires_grad_(), t["k"].requires_grad_()
    dq, dk = torch.autograd.grad(scene_attention(q, k, k, layout), (q, k), t["dout"])
    ref.close(dq, want["dq"], tol["dq"], "dq")
    both_ = want["dk"] + want["dv"]
    ref.close(dk, both_, tol["dk"] + tol["dv"] + (ref.ROUND[dt] + ref.U) * both_.abs(), "dk + dv")
    for narrow in (t["k"].detach()[:, :1], t["k"].detach()[:1]):
        leaf = narrow.clone().requires_grad_()
        got, = torch.autograd.grad(scene_attention(q, leaf.expand(75, 2, 16), t["v"], layout), leaf, t["dout"])
        want, tol = ref.attention(t["q"], narrow.expand(75, 2, 16), t["v"], seen, 0.25, 0.0, None, None, None, t["dout"])
        d = 1 if narrow.shape[1] == 1 else 0
        n = narrow.expand(75, 2, 16).shape[d]
        # torch adds the n gradients in fp32 (bf16: rounded once more at the end)
        ref.close(got, want["dk"].sum(d, keepdim=True), tol["dk"].sum(d, keepdim=True) + n * ref.U * want["dk"].abs().sum(d, keepdim=True)
                  + 2 * ref.ROUND[dt] * want["dk"].sum(d, keepdim=True).abs(), "spread")


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_offsets_beyond_32_bits(dt):
    """Rows 2^31 + 64 elements apart (the fourth one begins beyond 2^32 elements), and scenes of a cache 2^32 + 64 apart: the bits of the packed call."""
    n, H, KV, D, far = 4, 4, 2, 16, 2 ** 31 + 64
    t = inputs(4, n, n, H, KV, D, dt, 0)
    big = torch.empty(3 * far + 4096, dtype=dt, device=DEV)
    views, at = {}, 0
    for name, heads in (("q", H), ("k", KV), ("v", KV), ("dout", H)):
        views[name] = big.as_strided((n, heads, D), (far, D, 1), at)
        views[name].copy_(t[name])
        at += heads * D
    assert big.numel() > 2 ** 32

    def run(x):
        leaves = [x[m].detach().requires_grad_() for m in ("q", "k", "v")]
        out = scene_attention(*leaves, SceneLayout([0, n], causal=1))
        return (out,) + torch.autograd.grad(out, leaves, x["dout"])
    for a, b in zip(run(views), run(t)):
        assert torch.equal(a, b)
    axes, pos = RotaryAxes(D, (4, 4)), torch.rand((n, 2), device=DEV) * 50
    want = rotary(t["q"], t["k"], pos, axes)
    for a, b in zip(rotary(views["q"], views["k"], pos, axes), want):
        assert torch.equal(a, b)
    rotary(views["q"], views["k"], pos, axes, inplace=True)
    assert torch.equal(views["q"], want[0]) and torch.equal(views["k"], want[1])
    s = step_inputs(9, [2, 1], [700, 650], 700, H, KV, D, dt, 0)
    for name in ("k", "v"):
        c = big.as_strided((2, 700, KV, D), (2 ** 32 + 64, 2 * KV * D, D, 1), 0 if name == "k" else KV * D)
        c.copy_(s[name])
        views["c" + name] = c
    layout = SceneLayout(s["ptr"])
    assert torch.equal(scene_attention_step(s["q"], views["ck"], views["cv"], s["k_len"], layout), scene_attention_step(s["q"], s["k"], s["v"], s["k_len"], layout))
