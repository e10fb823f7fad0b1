"""GPU: attention over the rows of a scene and rotary positions against the 64-bit formulas (tests/scene_attn_ref.py), at the sizes, masks
and layouts where they can go wrong; tolerances are the bounds of the arithmetic computed there."""
import math

import numpy as np
import pytest
import torch

from dagnet_amd._capi import DagnetHipError
from dagnet_amd.attention import RotaryAxes, SceneLayout, rotary, scene_attention, scene_attention_step
from tests import scene_attn_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def randn(g, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dt).to(DEV)


def inputs(seed, nq, nk, H, KV, D, dt, axes):
    g = torch.Generator().manual_seed(seed)
    t = dict(q=randn(g, (nq, H, D), dt, 1.5), k=randn(g, (nk, KV, D), dt), v=randn(g, (nk, KV, D), dt), dout=randn(g, (nq, H, D), dt))
    t["slopes"] = (0.3 * torch.rand(H, generator=g) - 0.05).to(DEV) if axes else None
    t["pos"] = (torch.rand((nq, axes), generator=g) * 20).to(DEV) if axes else None
    t["k_pos"] = (torch.rand((nk, axes), generator=g) * 20).to(DEV) if axes else None
    return t


def both(t, layout, seen, cap=0.0, scale=None, same=False):
    """Kernel forward and backward against the formulas."""
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v")] + ([t["slopes"].requires_grad_()] if t["slopes"] is not None else [])
    kw = dict(pos=t["pos"], k_pos=None if same else t["k_pos"]) if t["slopes"] is not None else {}
    out = scene_attention(t["q"], t["k"], t["v"], layout, scale=scale, softcap=cap, slopes=t["slopes"], **kw)
    grads = torch.autograd.grad(out, leaves, t["dout"])
    want, tol = ref.attention(t["q"], t["k"], t["v"], seen, scale if scale is not None else t["q"].shape[2] ** -0.5, cap, t["slopes"], t["pos"],
                              t["pos"] if same else t["k_pos"], t["dout"])
    for name, got in zip(("out", "dq", "dk", "dv", "dslopes"), (out,) + grads):
        assert got.dtype == (F32 if name == "dslopes" else t["q"].dtype)
        ref.close(got, want[name], tol[name], name)
    return out, grads


LAYOUTS = {
    "one_row": ([0, 1], 0, 0),
    "one_scene": ([0, 10], 0, 0),
    "players": (list(range(0, 261, 10)), 0, 0),
    "ragged_and_empty": ([0, 1, 1, 18, 50, 51, 51, 53, 84, 101], 0, 0),
    "causal": ([0, 130], 1, 0),
    "causal_scenes": ([0, 7, 64, 65, 200], 1, 0),
    "steps_prefix": ([0, 60, 63, 135], [5, 3, 8], [20, 3, 0]),
    "prefix_longer_than_scene": ([0, 20, 90], 1, 40),
    "long": ([0, 333], [7], 31),
    "keys_in_parts": ([0, 1100], 1, 0),
    "two_in_parts": ([0, 1, 640, 1290], 0, 0),
    "prefix_in_parts": ([0, 1027], 9, 600),
}


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("name", list(LAYOUTS))
def test_layouts_forward_and_backward(name, dt):
    ptr, causal, prefix = LAYOUTS[name]
    t = inputs(len(name), ptr[-1], ptr[-1], 4, 2, 16, dt, 2)
    both(t, SceneLayout(ptr, causal=causal, prefix=prefix), ref.seen_matrix(ptr, None, causal, prefix), same=True)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [1, 3, 8, 16, 20, 33, 64, 72, 100, 127, 128])
def test_head_widths(D, dt):
    ptr = [0, 37, 100]
    t = inputs(D, 100, 100, 3, 3, D, dt, 0)
    both(t, SceneLayout(ptr, causal=1), ref.seen_matrix(ptr, None, 1))


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("H,KV", [(1, 1), (3, 1), (6, 3), (8, 2), (32, 1), (12, 4)])
def test_shared_heads(H, KV, dt):
    ptr = [0, 9, 70]
    t = inputs(H, 70, 70, H, KV, 40, dt, 1)
    both(t, SceneLayout(ptr, causal=3, prefix=4), ref.seen_matrix(ptr, None, 3, 4), cap=5.0, same=True)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("cap,axes", [(0.0, 0), (0.0, 1), (0.0, 3), (2.0, 0), (30.0, 2), (50.0, 3)])
def test_cap_and_distance(cap, axes, dt):
    ptr = [0, 80, 141]
    t = inputs(7, 141, 141, 2, 2, 32, dt, axes)
    both(t, SceneLayout(ptr, causal=2), ref.seen_matrix(ptr, None, 2), cap=cap, scale=0.7, same=True)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("q_ptr,k_ptr,causal", [([0, 5, 40], [0, 90, 90], 0), ([0, 5, 40], [0, 90, 200], 1), ([0, 50, 90], [0, 20, 60], 1),
                                                ([0, 0, 3], [0, 65, 70], 0), ([0, 30, 30], [0, 0, 70], 4)])
def test_other_rows_as_keys(q_ptr, k_ptr, causal, dt):
    """Rows without keys, keys without rows, causal rows before the first key."""
    t = inputs(11, q_ptr[-1], k_ptr[-1], 4, 2, 24, dt, 2)
    seen = ref.seen_matrix(q_ptr, k_ptr, causal)
    out, grads = both(t, SceneLayout(q_ptr, k_ptr, causal=causal), seen)
    dark = ~seen.any(1)
    assert (out[dark.to(DEV)] == 0).all() and (grads[0][dark.to(DEV)] == 0).all()


def test_no_rows_and_no_keys():
    t = inputs(1, 0, 30, 2, 2, 16, F32, 0)
    out, grads = both(t, SceneLayout([0, 0], [0, 30]), torch.zeros((0, 30), dtype=torch.bool))
    assert out.shape == (0, 2, 16) and (grads[1] == 0).all() and (grads[2] == 0).all()
    t = inputs(1, 30, 0, 2, 2, 16, F32, 0)
    out, grads = both(t, SceneLayout([0, 30], [0, 0]), torch.zeros((30, 0), dtype=torch.bool))
    assert (out == 0).all() and (grads[0] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_strided_views_and_expanded_gradients(dt):
    """q, k and v as slices of one product's output, at an odd element offset too; the gradient of a sum arrives expanded (strides 0)."""
    ptr = [0, 33, 75]
    N, H, KV, D = 75, 4, 2, 24
    for extra in (0, 1, 4):
        g = torch.Generator().manual_seed(extra)
        wide = randn(g, (N, (H + 2 * KV) * D + extra), dt)[:, extra:]
        q, k, v = (a.unflatten(1, (-1, D)) for a in wide.split([H * D, KV * D, KV * D], 1))
        t = dict(q=q.detach(), k=k.detach(), v=v.detach(), slopes=None, pos=None, k_pos=None, dout=randn(g, (N, H, D), dt))
        assert not t["q"].is_contiguous()
        both(t, SceneLayout(ptr), ref.seen_matrix(ptr))
    leaf = t["q"].contiguous().requires_grad_()
    a, = torch.autograd.grad(scene_attention(leaf, t["k"], t["v"], SceneLayout(ptr)).sum(), leaf)
    b, = torch.autograd.grad(scene_attention(leaf, t["k"], t["v"], SceneLayout(ptr)), leaf, torch.ones_like(leaf))
    assert torch.equal(a, b)
    c, = torch.autograd.grad(scene_attention(leaf, t["k"].transpose(1, 2).contiguous().transpose(1, 2), t["v"], SceneLayout(ptr)), leaf, torch.ones_like(leaf))
    assert torch.equal(a, c)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_places_do_not_reach_a_row(dt, bad):
    """NaN and infinities in the rows of one scene, and behind a causal bound: every other row and key keeps its bits."""
    ptr, H, KV, D = [0, 11, 14, 40], 4, 2, 20
    layout = SceneLayout(ptr, causal=[0, 0, 1])

    def run(t):
        leaves = [t[n].requires_grad_() for n in ("q", "k", "v")]
        o = scene_attention(*leaves, layout)
        return (o,) + torch.autograd.grad(o, leaves, t["dout"])
    clean = run(inputs(3, 40, 40, H, KV, D, dt, 0))
    for names in (("k", "v"), ("q", "dout"), ("q", "k", "v", "dout")):
        t = inputs(3, 40, 40, H, KV, D, dt, 0)
        for n in names:
            t[n][12] = bad                                        # one row of the second scene
        got = run(t)
        for a, b in zip(got, clean):
            keep = [i for i in range(40) if not 11 <= i < 14]
            if "k" in names:
                assert not torch.isfinite(got[0][11:14]).all()
            ref_t, ref_b = a[keep].float(), b[keep].float()
            assert torch.isfinite(ref_t).all()
            assert (ref_t - ref_b).abs().max() <= 2.0 ** (-7 if dt is BF16 else -18) * ref_b.abs().max()     # the slow form sums in another order
    t = inputs(3, 40, 40, H, KV, D, dt, 0)
    t["v"][39] = bad                                              # the last key of the causal scene: only its last row sees it
    got = run(t)
    assert torch.isfinite(got[0][:39].float()).all() and not torch.isfinite(got[0][39].float()).all()
    assert torch.isfinite(got[1][:39].float()).all()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_masked_places_in_long_rows_whose_keys_are_split(dt):
    N, H, D = 1100, 2, 24
    layout = SceneLayout([0, N], causal=1)

    def run(spoil):
        t = inputs(4, N, N, H, H, D, dt, 1)
        if spoil:
            t["k"][900], t["v"][900], t["q"][950], t["dout"][950] = float("nan"), float("inf"), float("inf"), float("nan")
        leaves = [t[n].requires_grad_() for n in ("q", "k", "v", "slopes")]
        o = scene_attention(t["q"], t["k"], t["v"], layout, slopes=t["slopes"], pos=t["pos"])
        return (o,) + torch.autograd.grad(o, leaves, t["dout"])
    clean, got = run(False), run(True)
    for a, b, n in zip(got[:2], clean[:2], ("out", "dq")):                      # rows before the spoilt key
        x, y = a[:900].float(), b[:900].float()
        assert torch.isfinite(x).all() and not torch.isfinite(a[900:].float()).all()
        assert (x - y).abs().max() <= 2.0 ** (-7 if dt is BF16 else -17) * y.abs().max(), n
    for a in got[2:4]:                                                          # keys behind the spoilt row are seen by fine rows alone, but for those
        assert torch.isfinite(a[951:].float()).all() == torch.isfinite(got[1][951:].float()).all()


def test_values_at_the_ends_of_the_type():
    """Scores far beyond exp's range, the type's lowest value as a key, and scores that all tie."""
    ptr = [0, 50]
    t = inputs(5, 50, 50, 2, 2, 16, F32, 0)
    t["q"] = t["q"] * 100
    t["k"] = t["k"] * 100
    both(t, SceneLayout(ptr), ref.seen_matrix(ptr))
    t = inputs(5, 50, 50, 2, 2, 16, F32, 0)
    t["k"][7] = torch.finfo(F32).min
    out = scene_attention(t["q"], t["k"], t["v"], SceneLayout(ptr), softcap=10.0)
    want, tol = ref.attention(t["q"], t["k"], t["v"], ref.seen_matrix(ptr), 0.25, 10.0)
    ref.close(out, want["out"], tol["out"].nan_to_num(0.0) + 1e-5, "saturated key")      # its score is +-10 whatever the sum's rounding
    t["q"].zero_()
    out = scene_attention(t["q"], t["k"][:, :, :].clamp(-1, 1), t["v"], SceneLayout(ptr))
    assert (out - t["v"].mean(0, keepdim=True)).abs().max() <= 64 * ref.U * t["v"].abs().max()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_gradients_repeat_and_match_differences(dt):
    ptr = [0, 45, 96]
    t = inputs(21, 96, 96, 4, 2, 32, dt, 2)
    layout, seen = SceneLayout(ptr, causal=3), ref.seen_matrix(ptr, None, 3)
    a = both(t, layout, seen, cap=20.0, same=True)
    b = both(t, layout, seen, cap=20.0, same=True)
    for x, y in zip((a[0],) + a[1], (b[0],) + b[1]):
        assert torch.equal(x, y)
    # central differences of the 64-bit formula along a random direction; h^2 of the third derivative is what is left
    g = torch.Generator().manual_seed(1)
    names = ("q", "k", "v", "slopes")
    dirs = [torch.randn(t[n].shape, generator=g, dtype=torch.float64) for n in names]

    def value(h):
        m = [t[n].detach().cpu().double() + h * d for n, d in zip(names, dirs)]
        x = {}
        for n, a_ in zip(names, m):
            x[n] = a_
        return _value64(x, t["pos"].cpu().double(), seen, 32 ** -0.5, 20.0, t["dout"].cpu().double())
    h = 1e-5
    slope = (value(h) - value(-h)) / (2 * h)
    got = sum(float((gr.detach().cpu().double() * d).sum()) for gr, d in zip(a[1], dirs))
    want, tol = ref.attention(t["q"], t["k"], t["v"], seen, 32 ** -0.5, 20.0, t["slopes"], t["pos"], t["pos"], t["dout"])
    room = sum(float((tol[n] * d.abs()).sum()) for n, d in zip(("dq", "dk", "dv", "dslopes"), dirs))
    assert abs(got - slope) <= room + 1e-6 * abs(slope) + 1e-6


def _value64(x, pos, seen, scale, cap, dout):
    H, KV = x["q"].shape[1], x["k"].shape[1]
    dist = (pos[:, None] - pos[None]).square().sum(-1).sqrt()
    tot = 0.0
    for h in range(H):
        c = h // (H // KV)
        z = cap * torch.tanh(x["q"][:, h] @ x["k"][:, c].t() * scale / cap) - x["slopes"][h] * dist
        o = torch.softmax(z.masked_fill(~seen, float("-inf")), 1) @ x["v"][:, c]
        tot = tot + (o * dout[:, h]).sum()
    return float(tot)


def test_only_what_is_asked_for_gets_a_gradient():
    ptr = [0, 30]
    t = inputs(2, 30, 30, 2, 2, 16, F32, 1)
    layout = SceneLayout(ptr)
    full = both(t, layout, ref.seen_matrix(ptr), same=True)[1]
    for i, n in enumerate(("q", "k", "v", "slopes")):
        x = {m: t[m].detach() for m in ("q", "k", "v", "slopes")}
        x[n].requires_grad_()
        out = scene_attention(x["q"], x["k"], x["v"], layout, slopes=x["slopes"], pos=t["pos"])
        got, = torch.autograd.grad(out, x[n], t["dout"])
        assert torch.equal(got, full[i])
    leaf = t["q"].detach().requires_grad_()
    g, = torch.autograd.grad(scene_attention(leaf, t["k"].detach(), t["v"].detach(), layout).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)                       # no second derivative: refused, not wrong


def test_default_positions_are_the_places_in_the_scene():
    ptr = [0, 40, 61]
    t = inputs(9, 61, 61, 2, 1, 16, F32, 1)
    at = torch.cat([torch.arange(40), torch.arange(21)]).float()[:, None].to(DEV)
    layout = SceneLayout(ptr, causal=1)
    assert torch.equal(scene_attention(t["q"], t["k"], t["v"], layout, slopes=t["slopes"]),
                       scene_attention(t["q"], t["k"], t["v"], layout, slopes=t["slopes"], pos=at))


# ---------------------------------------------------------------------------------------------------------------------
# a step over kept keys
# ---------------------------------------------------------------------------------------------------------------------
def step_inputs(seed, rows, lens, room, H, KV, D, dt, axes):
    g = torch.Generator().manual_seed(seed)
    S, N = len(lens), sum(rows)
    t = dict(q=randn(g, (N, H, D), dt, 1.5), k=randn(g, (S, room, KV, D), dt), v=randn(g, (S, room, KV, D), dt))
    t["k_len"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    t["slopes"] = (0.2 * torch.rand(H, generator=g)).to(DEV) if axes else None
    t["pos"] = (torch.rand((N, axes), generator=g) * 20).to(DEV) if axes else None
    t["k_pos"] = (torch.rand((S, room, axes), generator=g) * 20).to(DEV) if axes else None
    t["ptr"] = [0] + list(np.cumsum(rows))
    return t


def step_want(t, lens, cap, scale):
    """The cache's rows as one long batch of keys, most of them seen by nobody."""
    S, room = t["k"].shape[:2]
    seen = torch.zeros((t["q"].shape[0], S * room), dtype=torch.bool)
    for s in range(S):
        seen[t["ptr"][s]:t["ptr"][s + 1], s * room:s * room + lens[s]] = True
    flat = lambda x: None if x is None else x.flatten(0, 1)  # noqa: E731
    return ref.attention(t["q"], flat(t["k"]), flat(t["v"]), seen, scale, cap, t["slopes"], t["pos"], flat(t["k_pos"]))


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,lens,room,H,KV,D,axes,cap", [
    ([1], [1], 1, 1, 1, 16, 0, 0.0), ([10], [500], 500, 4, 4, 16, 2, 0.0), ([1, 1, 1], [0, 33, 700], 700, 8, 2, 64, 0, 30.0),
    ([3, 0, 17, 1], [64, 5, 1000, 999], 1024, 6, 3, 40, 3, 0.0), ([7, 10], [31, 2000], 2000, 12, 1, 128, 1, 20.0),
    ([5, 2], [129, 1], 300, 2, 2, 20, 0, 0.0), ([1, 2], [257, 511], 513, 3, 1, 7, 2, 0.0), ([40], [90], 100, 4, 1, 72, 0, 0.0)])
def test_step_over_kept_keys(rows, lens, room, H, KV, D, axes, cap, dt):
    t = step_inputs(room, rows, lens, room, H, KV, D, dt, axes)
    for s, n in enumerate(lens):                                   # what lies behind the kept keys is nobody's
        t["k"][s, n:], t["v"][s, n:] = float("nan"), float("inf")
    got = scene_attention_step(t["q"], t["k"], t["v"], t["k_len"], SceneLayout(t["ptr"]), softcap=cap, slopes=t["slopes"], pos=t["pos"], k_pos=t["k_pos"])
    for s, n in enumerate(lens):
        t["k"][s, n:], t["v"][s, n:] = 0.0, 0.0
    want, tol = step_want(t, lens, cap, D ** -0.5)
    ref.close(got, want["out"], tol["out"], "step")


def test_step_reads_a_cache_of_any_strides_and_clamps_its_lengths():
    t = step_inputs(4, [3, 2], [70, 41], 100, 4, 2, 32, BF16, 0)
    layout = SceneLayout(t["ptr"])
    want = scene_attention_step(t["q"], t["k"], t["v"], t["k_len"], layout)
    by_head = t["k"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    both_ = torch.stack([t["k"], t["v"]], 2)                        # [S, room, 2, KV, D]
    assert torch.equal(want, scene_attention_step(t["q"], by_head, t["v"], t["k_len"], layout))
    assert torch.equal(want, scene_attention_step(t["q"], both_[:, :, 0], both_[:, :, 1], t["k_len"], layout))
    far = torch.tensor([100000, -5], dtype=torch.int32, device=DEV)
    full = torch.tensor([100, 0], dtype=torch.int32, device=DEV)
    a, b = scene_attention_step(t["q"], t["k"], t["v"], far, layout), scene_attention_step(t["q"], t["k"], t["v"], full, layout)
    assert torch.equal(a, b) and (a[3:] == 0).all()


# ---------------------------------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------------------------------
def rotary_close(got, x, pos, axes, inverse=False):
    """|error| <= (4 u + r) of the pair's length: sine and cosine to 2 u, three operations, one rounding."""
    want = ref.turned(x, pos, axes.freq, axes.axis, axes.interleaved, inverse)
    P = axes.n_pairs
    i = torch.arange(P)
    a, b = (2 * i, 2 * i + 1) if axes.interleaved else (i, P + i)
    size = want.abs()
    size[..., a] = size[..., b] = (want[..., a].square() + want[..., b].square()).sqrt()
    tol = (6 * ref.U + ref.ROUND[x.dtype]) * size
    tol[..., 2 * P:] = 0.0
    ref.close(got, want, tol, "rotary")


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,H,KV,D,pairs,far", [(1, 1, 1, 2, (1,), 10), (10, 8, 2, 64, (12, 10, 10), 200), (33, 3, 1, 20, (3, 4), 1e6), (257, 4, 4, 17, (2, 1, 3), 1e4),
                                                (64, 16, 4, 128, (32, 16, 16), 1e6), (5, 2, 2, 80, (0, 40), 50), (19, 1, 1, 300, (100, 40), 100)])
def test_rotary_forward_and_backward(n, H, KV, D, pairs, far, interleaved, dt):
    g = torch.Generator().manual_seed(n)
    q, k = randn(g, (n, H, D), dt).requires_grad_(), randn(g, (n, KV, D), dt).requires_grad_()
    pos = (torch.rand((n, len(pairs)), generator=g) * 2 * far - far).to(DEV)
    axes = RotaryAxes(D, pairs, interleaved=interleaved)
    a, b = rotary(q, k, pos, axes)
    rotary_close(a, q, pos, axes), rotary_close(b, k, pos, axes)
    ga, gb = randn(g, (n, H, D), dt), randn(g, (n, KV, D), dt)
    da, db = torch.autograd.grad((a, b), (q, k), (ga, gb))
    rotary_close(da, ga, pos, axes, True), rotary_close(db, gb, pos, axes, True)


@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_rotary_of_whole_positions_views_and_in_place(dt):
    g = torch.Generator().manual_seed(0)
    wide = randn(g, (21, 6 * 32 + 3), F32)[:, 3:]
    q, k = wide[:, :4 * 32].unflatten(1, (4, 32)), wide[:, 4 * 32:].unflatten(1, (2, 32))
    pos = torch.randint(-2 ** 30, 2 ** 30, (21, 2), generator=g).to(dt).to(DEV)
    axes = RotaryAxes(32, (8, 8), theta=(10000.0, 100.0))
    a, b = rotary(q, k, pos, axes)
    rotary_close(a, q, pos, axes), rotary_close(b, k, pos, axes)
    only, none = rotary(q, None, pos, axes)
    assert none is None and torch.equal(only, a)
    x, y = rotary(q, k, pos, axes, inplace=True)
    assert x is q and y is k and torch.equal(q, a) and torch.equal(k, b)
    e, f = rotary(q[:0], k[:0], pos[:0], axes)
    assert e.shape == (0, 4, 32) and f.shape == (0, 2, 32)


# ---------------------------------------------------------------------------------------------------------------------
# together, streams, graphs
# ---------------------------------------------------------------------------------------------------------------------
def test_a_rollout_step_by_step_equals_the_whole_sequence():
    """Rotary positions, the whole sequence at once (causal by time step), and the same one time step after the other over a cache."""
    agents, T, H, KV, D, cap = [3, 5, 1], 6, 4, 2, 32, 15.0
    S, room = 3, 5 * T
    rows = [a * T for a in agents]
    ptr = [0] + list(np.cumsum(rows))
    N = ptr[-1]
    g = torch.Generator().manual_seed(8)
    q, k, v = randn(g, (N, H, D), F32), randn(g, (N, KV, D), F32), randn(g, (N, KV, D), F32)
    when = torch.cat([torch.arange(T).repeat_interleave(a) for a in agents]).float()
    pos = torch.cat([when[:, None], torch.rand((N, 2), generator=g) * 50], 1).to(DEV)
    axes, slopes = RotaryAxes(D, (8, 4, 4), device=DEV), torch.tensor([0.5, 0.1, 0.02, 0.0], device=DEV)
    qr, kr = rotary(q, k, pos, axes)
    whole = scene_attention(qr, kr, v, SceneLayout(ptr, causal=agents), softcap=cap, slopes=slopes, pos=pos)
    kc, vc, pc = torch.zeros((S, room, KV, D), device=DEV), torch.zeros((S, room, KV, D), device=DEV), torch.zeros((S, room, 3), device=DEV)
    k_len = torch.zeros(S, dtype=torch.int32, device=DEV)
    layout = SceneLayout([0] + list(np.cumsum(agents)), device=DEV)
    for t in range(T):
        rows_t = torch.cat([torch.arange(ptr[s] + t * a, ptr[s] + (t + 1) * a) for s, a in enumerate(agents)]).to(DEV)
        slot = torch.cat([torch.arange(s * room + t * a, s * room + (t + 1) * a) for s, a in enumerate(agents)]).to(DEV)
        a_, b_ = rotary(q[rows_t], k[rows_t], pos[rows_t], axes)
        kc.view(-1, KV, D).index_copy_(0, slot, b_)
        vc.view(-1, KV, D).index_copy_(0, slot, v[rows_t])
        pc.view(-1, 3).index_copy_(0, slot, pos[rows_t])
        k_len.copy_(torch.tensor([(t + 1) * a for a in agents], dtype=torch.int32))
        got = scene_attention_step(a_, kc, vc, k_len, layout, softcap=cap, slopes=slopes, pos=pos[rows_t], k_pos=pc)
        assert (got - whole[rows_t]).abs().max() <= 2e-5 * whole.abs().max()      # two orders of the same fp32 sums


def _chain(t, layout, axes, rp):
    leaves = [t[n] for n in ("q", "k", "v", "slopes")]
    a, b = rotary(t["q"], t["k"], rp, axes)
    o = scene_attention(a, b, t["v"], layout, softcap=10.0, slopes=t["slopes"], pos=t["pos"])
    return (o,) + torch.autograd.grad(o, leaves, t["dout"])


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_replays_of_a_captured_training_pass(dt):
    """Two graphs of the same calls, replayed in turn with eager work between, on inputs that change: every replay equals the eager call."""
    ptr = [0, 45, 100]
    t = inputs(31, 100, 100, 4, 2, 32, dt, 2)
    for n in ("q", "k", "v", "slopes"):
        t[n].requires_grad_()
    layout, axes = SceneLayout(ptr, causal=5, device=DEV), RotaryAxes(32, (8, 8), device=DEV)
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _chain(t, layout, axes, t["pos"])
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _chain(t, layout, axes, t["pos"])
        graphs.append((g, out))
    for i in range(4):
        with torch.no_grad():
            t["q"].mul_(0.9)
            t["pos"].add_(1.5)
        want = [x.clone() for x in _chain(t, layout, axes, t["pos"])]
        torch.cuda.synchronize()
        for g, out in graphs:
            g.replay()
            want2 = _chain(t, layout, axes, t["pos"])
            torch.cuda.synchronize()
            for a, b, c in zip(out, want, want2):
                assert torch.equal(a, b) and torch.equal(b, c)


def test_replays_of_a_captured_step_follow_the_cache():
    t = step_inputs(6, [4, 4], [600, 300], 1200, 8, 2, 64, BF16, 3)
    layout = SceneLayout(t["ptr"], device=DEV)
    run = lambda: scene_attention_step(t["q"], t["k"], t["v"], t["k_len"], layout, slopes=t["slopes"], pos=t["pos"], k_pos=t["k_pos"])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = run()
    with torch.cuda.graph(g2):
        o2 = run()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for n in ([601, 1200], [1, 0], [1199, 640]):
        t["k_len"].copy_(torch.tensor(n, dtype=torch.int32))
        want = run().clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):                                # two graphs in flight at once: their workspaces are their own
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, want) and torch.equal(o2, want)


def test_calls_on_several_streams_at_once():
    ptr = [0, 300, 800]
    layout = SceneLayout(ptr, causal=1)
    ts = [inputs(s, 800, 800, 4, 2, 64, BF16, 0) for s in range(3)]
    want = [_plain_run(t, layout) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ts]
    outs = []
    for _ in range(3):
        for t, s in zip(ts, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(_plain_run(t, layout))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        for a, b in zip(o, want[i % 3]):
            assert torch.equal(a, b)


def _plain_run(t, layout):
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v")]
    o = scene_attention(*leaves, layout)
    return (o.detach(),) + torch.autograd.grad(o, leaves, t["dout"])


def test_tables_are_not_uploaded_into_a_capture():
    t = inputs(1, 20, 20, 2, 2, 16, F32, 0)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(DagnetHipError, match="before capturing"), torch.cuda.graph(g):
        scene_attention(t["q"], t["k"], t["v"], SceneLayout([0, 20]))
    del g
    torch.cuda.synchronize()


def test_mixed_devices_are_refused():
    t = inputs(1, 20, 20, 2, 2, 16, F32, 1)
    with pytest.raises(DagnetHipError, match="ROCm device"):
        scene_attention(t["q"], t["k"].cpu(), t["v"], SceneLayout([0, 20]))
    with pytest.raises(DagnetHipError, match="ROCm device"):
        scene_attention(t["q"], t["k"], t["v"], SceneLayout([0, 20]), slopes=t["slopes"], pos=t["pos"].cpu())


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("names", [("q",), ("slopes",), ("q", "slopes"), ("k", "v")])
def test_rows_repaired_one_by_one_whichever_gradients_are_wanted(names, dt):
    """A NaN in a key of another scene sends the rows of its tile through the form that takes them one by one; what that form reads has to be there
    (memory that the calls get is filled with large values first)."""
    ptr = [0, 20, 51]
    t = inputs(5, 51, 51, 4, 2, 24, dt, 2)
    t["k"][22], t["v"][22] = float("nan"), float("nan")
    del t["k_pos"]
    layout = SceneLayout(ptr)
    leaves = [t[n].requires_grad_() for n in names]
    out = scene_attention(t["q"], t["k"], t["v"], layout, softcap=8.0, slopes=t["slopes"], pos=t["pos"])
    keep = [torch.full((n,), 1e4, device=DEV) for n in (64, 512, 4096, 1 << 16, 1 << 20) for _ in range(8)]
    del keep
    dout = t["dout"].clone()
    dout[20:] = 0
    got = dict(zip(names, torch.autograd.grad(out, leaves, dout)))
    cut = {n: t[n].detach()[:20] for n in ("q", "k", "v", "pos")}
    want, tol = ref.attention(cut["q"], cut["k"], cut["v"], ref.seen_matrix([0, 20], None, 0), 24 ** -0.5, 8.0, t["slopes"].detach(), cut["pos"], cut["pos"], t["dout"][:20])
    ref.close(out[:20], want["out"], tol["out"], "out")
    for n, g in got.items():
        if n == "slopes":
            assert g.isnan().all()                    # the other scene's own NaN
        else:
            ref.close(g[:20], want["d" + n], tol["d" + n], "d" + n)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_a_cap_far_below_the_scores(dt):
    t = inputs(9, 70, 70, 2, 1, 16, dt, 0)
    both(t, SceneLayout([0, 70], causal=1), ref.seen_matrix([0, 70], None, 1), cap=1e-3)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_a_cap_far_above_the_scores_is_none(dt):
    """cap 1e12 moves a score x by x^3 / 3e24.  tanh near zero is a product, a quotient and the two factors: at most six roundings, 6 U |x|, which
    is what the bounds without a cap hold for x already (2 U and 4 U of its size): twice those bounds."""
    t = inputs(9, 70, 70, 2, 1, 16, dt, 0)
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v")]
    out = scene_attention(*leaves, SceneLayout([0, 70], causal=1), softcap=1e12)
    want, tol = ref.attention(*leaves, ref.seen_matrix([0, 70], None, 1), 0.25, 0.0, None, None, None, t["dout"])
    for name, got in zip(("out", "dq", "dk", "dv"), (out,) + torch.autograd.grad(out, leaves, t["dout"])):
        ref.close(got, want[name], 2 * tol[name], name)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_a_cap_next_to_zero_gives_the_mean(dt):
    """Scores within 1e-12 of each other: p is 1 / n to eps, for rows of zeros too (0 / cap).  n = 40 terms: sums off by at most 40 eps of the values'
    size, the quotient, p's rounding (bf16: half a step, 2^-8) and the output's on top."""
    t = inputs(9, 40, 40, 2, 1, 16, dt, 0)
    t["q"][::2] = 0
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v")]
    out = scene_attention(*leaves, SceneLayout([0, 40]), softcap=1e-12)
    want = t["v"].detach().double().mean(0, keepdim=True).expand(40, 2, 16)
    size = t["v"].detach().double().abs().max().item()
    tol = size * 48 * 2 ** -23 + (size * 2 * 2 ** -8 if dt == BF16 else 0)
    assert ((out.double() - want).abs() <= tol).all()
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(out, leaves, t["dout"]))


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_positions_whose_squares_overflow(dt):
    """The far half is infinitely far in fp32 (2e20 ** 2 > 3.4e38): its keys have p = 0, as in 64 bits (exp(-0.1 2e20))."""
    t = inputs(3, 60, 60, 2, 2, 16, dt, 2)
    t["slopes"] = torch.full((2,), 0.1, device=DEV)
    near = t["pos"].clone()
    t["pos"][30:] += 2e20
    out = scene_attention(t["q"], t["k"], t["v"], SceneLayout([0, 60]), slopes=t["slopes"], pos=t["pos"])
    cut = {n: t[n][:30] for n in ("q", "k", "v")}
    want, tol = ref.attention(cut["q"], cut["k"], cut["v"], ref.seen_matrix([0, 30], None, 0), 0.25, 0.0, t["slopes"], near[:30], near[:30], t["dout"][:30])
    ref.close(out[:30], want["out"], tol["out"], "out")


@pytest.mark.parametrize("N", [700, 2500])
def test_a_batch_of_nan_gives_nan(N):
    """Every row is taken one by one then, and ends at its first key."""
    t = inputs(2, N, N, 4, 2, 32, BF16, 0)
    t["q"].fill_(float("nan"))
    leaves = [t[n].requires_grad_() for n in ("q", "k", "v")]
    out = scene_attention(*leaves, SceneLayout([0, N], causal=1))
    assert out.isnan().all() and all(g.isnan().all() for g in torch.autograd.grad(out, leaves, t["dout"]))


def test_in_place_rotary_is_seen_by_autograd():
    g = torch.Generator().manual_seed(1)
    q, k = randn(g, (9, 2, 16), F32), randn(g, (9, 2, 16), F32)
    axes, pos = RotaryAxes(16, (8,)), torch.arange(9, device=DEV)[:, None]
    w = torch.ones(16, device=DEV, requires_grad=True)
    before = (q * w).sum() + (k * w).sum()
    with torch.no_grad():
        rotary(q, k, pos, axes, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        before.backward()


def test_in_place_rotary_of_one_product_and_positions_within():
    """q and k as parts of one tensor, the positions another part of it; what is not turned stays."""
    g = torch.Generator().manual_seed(2)
    x = randn(g, (33, 5, 16), F32)
    pos = x[:, 4, :2]
    axes = RotaryAxes(16, (4, 4))
    was = x.clone()
    want = rotary(was[:, :2], was[:, 2:3], was[:, 4, :2], axes)
    rotary(x[:, :2], x[:, 2:3], pos, axes, inplace=True)
    assert torch.equal(x[:, :2], want[0]) and torch.equal(x[:, 2:3], want[1]) and torch.equal(x[:, 3:], was[:, 3:])
    rotary(x[:, :2], x[:, 4:], pos, axes, inplace=True)              # k holds the positions
    twice = rotary(want[0], was[:, 4:], was[:, 4, :2], axes)
    assert torch.equal(x[:, :2], twice[0]) and torch.equal(x[:, 4:], twice[1])


@pytest.mark.parametrize("which", [0, 1])
def test_one_of_the_two_turned_tensors_used(which):
    g = torch.Generator().manual_seed(3)
    q, k = randn(g, (17, 3, 16), F32).requires_grad_(), randn(g, (17, 1, 16), F32).requires_grad_()
    axes, pos = RotaryAxes(16, (5, 3)), torch.rand((17, 2), generator=g).to(DEV)
    out = rotary(q, k, pos, axes)[which]
    got = torch.autograd.grad(out.sum(), (q, k), allow_unused=True)
    alone = (q, k)[which].detach().requires_grad_()
    want = torch.autograd.grad(rotary(alone, None, pos, axes)[0].sum(), alone)[0]
    assert torch.equal(got[which], want) and (got[1 - which] is None or (got[1 - which] == 0).all())


def test_second_derivatives_are_refused_whatever_asks_for_them():
    t = inputs(4, 20, 20, 2, 2, 16, F32, 1)
    for names in (("q",), ("slopes",), ("q", "k", "v", "slopes")):
        leaves = [t[n].detach().requires_grad_() for n in names]
        a = {**t, **dict(zip(names, leaves))}
        out = scene_attention(a["q"], a["k"], a["v"], SceneLayout([0, 20]), slopes=a["slopes"], pos=a["pos"])
        grads = torch.autograd.grad(out.square().sum(), leaves, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            sum(x.sum() for x in grads).backward()


@pytest.mark.parametrize("H,KV,D,causal,cap,axes", [(72, 72, 64, 0, 0.0, 1), (72, 72, 72, 0, 20.0, 0), (128, 64, 128, 3, 20.0, 1), (128, 128, 33, 1, 0.0, 0)])
def test_rows_that_fill_the_chip(H, KV, D, causal, cap, axes):
    """bf16, enough (row, key head) tiles for two blocks of 16 rows a wave; ragged ends, a scene of one row, an empty one."""
    ptr = [0, 300, 301, 301, 800]
    t = inputs(D, 800, 800, H, KV, D, BF16, axes)
    both(t, SceneLayout(ptr, causal=causal), ref.seen_matrix(ptr, None, causal), cap=cap, same=True)
    with torch.no_grad():
        kw = dict(slopes=t["slopes"], pos=t["pos"]) if axes else {}
        out = scene_attention(t["q"], t["k"], t["v"], SceneLayout(ptr, causal=causal), softcap=cap, **kw)
    want, tol = ref.attention(t["q"], t["k"], t["v"], ref.seen_matrix(ptr, None, causal), D ** -0.5, cap, t["slopes"], t["pos"], t["pos"])
    ref.close(out, want["out"], tol["out"], "out")
