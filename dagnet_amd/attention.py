"""Dot-product attention over the rows of a scene, and rotary positions with several axes: what a model needs that replaces or follows
the graph layers (gat.py, gcn.py) by attention over a scene's agents, or over its agents by time steps.

    layout = SceneLayout(seq_start_end)                       # every agent of a scene sees every other
    layout = SceneLayout(scene_ptr, causal=agents, prefix=[a * obs_len for a in agents])   # whole sequences, time step after time step
    axes = RotaryAxes(head_dim, (16, 8, 8))                   # pairs of columns turned by time, y and x
    q, k = rotary(q, k, pos, axes)
    out = scene_attention(q, k, v, layout, softcap=30.0, slopes=slopes, pos=pos)           # differentiable
    out = scene_attention_step(q, k_cache, v_cache, k_len, step_layout)                    # the new rows of a rollout's step

The kernels are csrc/scene_attn_*.hip and csrc/rotary.hip behind dagnet_op_attn_* and dagnet_op_rotary (include/dagnet_hip.h), called
by csrc/torch_calls.cpp.  fp32 and bf16; there is no CPU path.  Calls are eager or captured into a graph: tracing, forward-mode derivatives and
function transforms are refused.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import numpy as np
import torch

from . import _ops
from ._capi import DagnetHipError

_TYPES = (torch.float32, torch.bfloat16)
_POSITIONS = (torch.float32, torch.int32, torch.int64)


class _Tables:
    """Small host tables that are uploaded once per device (before a graph capture: a capturing stream refuses the copy).  A captured
    graph replays with their addresses: keep the object as long as the graph."""

    def __init__(self):
        self._dev = {}

    def __getstate__(self):               # a copy (deepcopy, pickle) uploads its own: the addresses are this object's
        return {**self.__dict__, "_dev": {}}

    def _host(self) -> torch.Tensor:      # pragma: no cover - overridden
        raise NotImplementedError

    def _addresses(self, t: torch.Tensor) -> tuple:      # pragma: no cover - overridden
        raise NotImplementedError

    def tables(self, index: int) -> tuple:
        """-> the addresses of the tables on device ``index``, and the tensor that holds them."""
        got = self._dev.get(index)
        stream = _ops._raw_stream(index)
        if got is None:
            if torch.cuda.is_current_stream_capturing():
                raise DagnetHipError(f"{type(self).__name__}: make it with device=, or call it once, before capturing a graph")
            _ops.calls().eager()                                                 # a fake upload would be kept for later calls
            t = self._host().to(torch.device("cuda", index))
            got = self._dev[index] = (self._addresses(t) + (t,), stream)
        elif got[1] != stream:
            got[0][-1].record_stream(torch.cuda.current_stream(index))       # its memory is not handed on while a kernel of this stream may read it
        return got[0]


def _device(device) -> torch.device:
    d = torch.device(device)
    if d.type != "cuda":
        raise DagnetHipError(f"the HIP path needs a ROCm device and has no CPU fallback (got {d})")
    return d if d.index is not None else torch.device("cuda", torch.cuda.current_device())


def _ptr_of(ptr, what) -> np.ndarray:
    """[S + 1] row pointer, or the reference's seq_start_end [S, 2] -> int64 [S + 1].  Scenes may be empty."""
    p = ptr.detach().cpu().numpy() if isinstance(ptr, torch.Tensor) else np.asarray(ptr)
    if p.dtype.kind not in "iu":
        raise DagnetHipError(f"{what} must hold whole numbers, got {p.dtype}")
    p = p.astype(np.int64)
    if p.ndim == 2 and p.shape[1] == 2:
        if p.shape[0] < 1 or np.any(p[1:, 0] != p[:-1, 1]):
            raise DagnetHipError(f"{what}: scenes must follow each other without gaps")
        p = np.concatenate([p[:, 0], p[-1:, 1]])
    if p.ndim != 1 or p.shape[0] < 2 or p[0] != 0 or np.any(p[1:] < p[:-1]):
        raise DagnetHipError(f"{what} must be [S + 1] row pointers from 0 that do not decrease (or seq_start_end [S, 2])")
    if p[-1] > 0x7fff0000:
        raise DagnetHipError(f"{what}: {int(p[-1])} rows are too many for one batch")
    return p


def _per_scene(v, S, what) -> np.ndarray:
    a = v.detach().cpu().numpy() if isinstance(v, torch.Tensor) else np.asarray(v)
    if a.dtype.kind not in "iu" or a.ndim > 1 or (a.ndim == 1 and a.shape[0] != S):
        raise DagnetHipError(f"{what} must be one whole number, or one per scene ({S})")
    if np.any(a < 0):
        raise DagnetHipError(f"{what} must not be negative")
    return np.broadcast_to(a.astype(np.int64), (S,))


class SceneLayout(_Tables):
    """Which keys every row sees, for one batch layout (make it once and keep it, like a plan).

    ``ptr``: scene s owns query rows ptr[s] .. ptr[s + 1] - 1 (or the reference's seq_start_end); ``k_ptr``: the same for the keys when
    they are other rows (default: rows and keys are the same).  A row sees keys of its own scene only:
      * causal 0: all of them;
      * causal g: rows stand in groups of g (the agents of one time step; 1: plain sequences) and see up to the end of their own group;
        with more keys than rows the rows are the last ones of the sequence.  One number, or one per scene;
      * prefix p: with ``causal``, the first p keys of the scene are seen by all its rows (the observed steps).  One number, or one per scene.
    A scene without keys, or a causal row before the first key, sees nothing: its output is 0."""

    def __init__(self, ptr, k_ptr=None, *, causal: Union[int, Sequence[int]] = 0, prefix: Union[int, Sequence[int]] = 0, device=None):
        super().__init__()
        q = _ptr_of(ptr, "ptr")
        k = q if k_ptr is None else _ptr_of(k_ptr, "k_ptr")
        S = q.shape[0] - 1
        if k.shape[0] != S + 1:
            raise DagnetHipError(f"ptr has {S} scenes but k_ptr {k.shape[0] - 1}")
        group, pre = _per_scene(causal, S, "causal"), _per_scene(prefix, S, "prefix")
        if np.any((group == 0) & (pre > 0)):
            raise DagnetHipError("prefix needs causal: without it every row sees the whole scene")
        self.S, self.nq, self.nk, self.same_rows = S, int(q[-1]), int(k[-1]), k_ptr is None
        self.masked = bool(np.any(group > 0))
        n_q, n_k = np.diff(q), np.diff(k)
        self.max_rows = int(n_q.max()) if S else 0
        scene = np.repeat(np.arange(S), n_q)
        at = np.arange(self.nq) - q[scene] + (n_k - n_q)[scene]                 # the row's place among the scene's keys
        g = np.maximum(group[scene], 1)
        end = np.where(group[scene] > 0, np.maximum((at // g + 1) * g, pre[scene]), n_k[scene])
        lo = k[scene]
        hi = lo + np.clip(end, 0, n_k[scene])
        self.span = (int((hi - lo).max()), int((hi - lo).mean())) if self.nq else (0, 0)        # keys that a row sees: most, mean
        keys = np.arange(self.nk)
        self._tab = np.concatenate([lo, hi, np.searchsorted(hi, keys, side="right"), np.searchsorted(lo, keys, side="right"), q, k]).astype(np.int32)
        self._at, self._k_at = at, keys - np.repeat(k[:-1], n_k)
        self.far = bool(np.any(np.maximum(n_q, n_k) > 1 << 24))                 # a place may be no fp32 number
        if device is not None:
            self.tables(_device(device).index)

    def row_bounds(self):
        """-> (lo, hi): int32 arrays; row i sees the keys lo[i] <= j < hi[i]."""
        return self._tab[:self.nq], self._tab[self.nq:2 * self.nq]

    def _host(self):
        return torch.from_numpy(np.concatenate([self._tab, self._at.astype(np.float32).view(np.int32), self._k_at.astype(np.float32).view(np.int32)]))

    def _addresses(self, t):
        p, n, m = t.data_ptr(), 4 * self.nq, 4 * self.nk
        return p, p + n, p + 2 * n, p + 2 * n + m, p + 2 * n + 2 * m, self.span          # row_lo, row_hi, key_lo, key_hi, ptr

    def places(self, index):
        """-> fp32 [nq, 1], [nk, 1]: the places of rows and keys in their scenes, on device ``index``."""
        if self.far:
            raise DagnetHipError("places in a scene of more than 2^24 rows or keys are no fp32 numbers: pass pos (and k_pos)")
        t = self.tables(index)[-1][len(self._tab):].view(torch.float32)
        return t[:self.nq, None], t[self.nq:, None]


def _matrix3(t, what):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise DagnetHipError(f"{what} must be [rows, heads, head_dim]" + (f", got {tuple(t.shape)}" if isinstance(t, torch.Tensor) else ""))


def _columns(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_heads(q, k, v):
    dt = q.dtype
    if dt not in _TYPES or k.dtype is not dt or v.dtype is not dt:
        raise DagnetHipError(f"q, k and v must all be fp32 or all bf16 (got {q.dtype}, {k.dtype}, {v.dtype})")
    _, H, D = q.shape
    if not 1 <= D <= 128:
        raise DagnetHipError(f"head_dim must be 1 .. 128, got {D}")
    if k.shape != v.shape or k.shape[-1] != D:
        raise DagnetHipError(f"k and v must have one shape and q's head_dim {D}, got {tuple(k.shape)}, {tuple(v.shape)}")
    if H < 1 or k.shape[-2] < 1 or H % k.shape[-2]:
        raise DagnetHipError(f"{H} heads are no multiple of {k.shape[-2]} key heads")


def _check_device(names, *tensors) -> int:
    """-> the device index that all of them share."""
    index = tensors[0].get_device()
    for i, t in enumerate(tensors):
        if t is not None and (index < 0 or t.get_device() != index):
            raise DagnetHipError(f"{names.split()[i]} lives on {t.device}; every tensor must live on q's ROCm device ({tensors[0].device}); there is no CPU path")
    return index


def _numbers(scale, softcap, D):
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    softcap = float(softcap or 0.0)
    if not abs(scale) <= 1e15 or not (softcap == 0.0 or 1e-15 <= softcap <= 1e15):
        raise DagnetHipError(f"softcap must be 0 or 1e-15 .. 1e15 and scale within 1e15 (got scale {scale}, softcap {softcap})")
    return scale, softcap


def _check_slopes(slopes, H):
    if slopes.dtype != torch.float32 or tuple(slopes.shape) != (H,):
        raise DagnetHipError(f"slopes must be fp32 [{H}], got {slopes.dtype} {tuple(slopes.shape)}")


def _positions(p, lead, what):
    if not isinstance(p, torch.Tensor) or p.dtype != torch.float32 or p.dim() != len(lead) + 1 or tuple(p.shape[:-1]) != tuple(lead) or not 1 <= p.shape[-1] <= 3:
        raise DagnetHipError(f"{what} must be fp32 {list(lead) + ['1 .. 3']}" + (f", got {p.dtype} {tuple(p.shape)}" if isinstance(p, torch.Tensor) else ""))
    if p.requires_grad and torch.is_grad_enabled():
        raise DagnetHipError(f"{what}: positions have no gradient here; pass {what}.detach()")
    return p.contiguous()


def scene_attention(q, k, v, layout: SceneLayout, *, scale: Optional[float] = None, softcap: float = 0.0, slopes=None, pos=None, k_pos=None):
    """softmax_j(softcap tanh(scale q_i.k_j / softcap) - slopes_h |pos_i - k_pos_j|) v_j over the keys that ``layout`` lets row i see.

    q [nq, heads, head_dim], k and v [nk, key heads, head_dim] (head h reads key head h // (heads // key heads)), fp32 or bf16 with any row
    and head strides -> [nq, heads, head_dim].  scale: default head_dim ** -0.5.  softcap 0: scores are not capped.  slopes fp32 [heads]:
    decay of a score with the Euclidean distance of the rows' positions, pos [nq, 1 .. 3] fp32 (k_pos [nk, ..]: default pos where rows
    and keys are the same); without pos the distance is that of the rows' places in their scene (scenes of at most 2^24 rows and keys).  Differences of
    positions stay below 1e19: their squares leave fp32 beyond, such a key has no weight for a positive slope, and a slope of 0 and the slopes' gradient give NaN.
    Differentiable in q, k, v and slopes; gradients repeat bit for bit.  A row that sees nothing gives 0; what stands in keys a row does
    not see (infinities and NaN included) does not reach it.  fp32: fp32 products and sums.  bf16: fp32 scores and statistics, the
    probabilities (and their gradients) are rounded to bf16 for the second product, the output once at the end; where gradients are wanted the forward takes the
    probabilities as two bf16 terms (its output may differ in the last bit from a call without).
    A captured graph replays with the layout's tables: keep the layout as long as the graph."""
    if not isinstance(layout, SceneLayout):
        raise DagnetHipError("layout must be a SceneLayout")
    _matrix3(q, "q"), _matrix3(k, "k"), _matrix3(v, "v")
    _check_heads(q, k, v)
    if q.shape[0] != layout.nq or k.shape[0] != layout.nk:
        raise DagnetHipError(f"the layout has {layout.nq} rows and {layout.nk} keys, q has {q.shape[0]} and k {k.shape[0]}")
    scale, softcap = _numbers(scale, softcap, q.shape[2])
    if slopes is None:
        if pos is not None or k_pos is not None:
            raise DagnetHipError("positions without slopes have no effect: pass slopes")
    else:
        _check_slopes(slopes, q.shape[1])
        if pos is not None:
            pos = _positions(pos, (layout.nq,), "pos")
            if k_pos is None:
                if not layout.same_rows:
                    raise DagnetHipError("k_pos is missing: the keys are other rows than the queries")
                k_pos = pos
            else:
                k_pos = _positions(k_pos, (layout.nk,), "k_pos")
            if k_pos.shape[-1] != pos.shape[-1]:
                raise DagnetHipError(f"pos has {pos.shape[-1]} axes and k_pos {k_pos.shape[-1]}")
        elif k_pos is not None:
            raise DagnetHipError("k_pos without pos")
    index = _check_device("q k v slopes pos k_pos", q, k, v, slopes, pos, k_pos)
    if slopes is not None:
        slopes = slopes.contiguous()
        if pos is None:
            pos, k_pos = layout.places(index)
    return _ops.calls().scene_attn(_columns(q), _columns(k), _columns(v), slopes, layout.tables(index), scale, softcap, pos, k_pos)


def scene_attention_step(q, k_cache, v_cache, k_len, layout: SceneLayout, *, scale: Optional[float] = None, softcap: float = 0.0, slopes=None,
                         pos=None, k_pos=None):
    """The same attention for the new rows of a step over kept keys: row i of scene s (``layout`` names the scenes' rows) sees the first
    k_len[s] keys of k_cache[s].

    q [nq, heads, head_dim]; k_cache, v_cache [S, room, key heads, head_dim] with any strides but the last; k_len int32 [S] ON THE DEVICE (a
    captured call follows a growing cache; values are clamped to 0 .. room); pos [nq, 1 .. 3] and k_pos [S, room, ..] with slopes.  Write
    the new rows' own keys into the cache first if they are to see each other.  What stands behind k_len does not matter; an infinity or NaN in
    a key that is seen may make its rows not finite.  Roundings as in scene_attention without gradients.  No gradient.  -> [nq, heads, head_dim]."""
    if not isinstance(layout, SceneLayout):
        raise DagnetHipError("layout must be a SceneLayout")
    if layout.masked or not layout.same_rows:
        raise DagnetHipError("a step's layout names the new rows only (no k_ptr, causal or prefix): they see k_len keys of their scene")
    _matrix3(q, "q")
    if not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor) or k_cache.dim() != 4 or v_cache.dim() != 4:
        raise DagnetHipError("k_cache and v_cache must be [scenes, room, key heads, head_dim]")
    _check_heads(q, k_cache, v_cache)
    S, room = k_cache.shape[:2]
    if q.shape[0] != layout.nq or S != layout.S:
        raise DagnetHipError(f"the layout has {layout.nq} rows in {layout.S} scenes, q has {q.shape[0]} rows and the cache {S} scenes")
    if not isinstance(k_len, torch.Tensor) or k_len.dtype != torch.int32 or tuple(k_len.shape) != (S,):
        raise DagnetHipError(f"k_len must be int32 [{S}]")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k_cache, v_cache, slopes)):
        raise DagnetHipError("scene_attention_step has no gradient: call it under torch.no_grad(), or use scene_attention")
    scale, softcap = _numbers(scale, softcap, q.shape[2])
    if slopes is None:
        if pos is not None or k_pos is not None:
            raise DagnetHipError("positions without slopes have no effect: pass slopes")
    else:
        _check_slopes(slopes, q.shape[1])
        pos, k_pos = _positions(pos, (layout.nq,), "pos"), _positions(k_pos, (S, room), "k_pos")
        if k_pos.shape[-1] != pos.shape[-1]:
            raise DagnetHipError(f"pos has {pos.shape[-1]} axes and k_pos {k_pos.shape[-1]}")
        slopes = slopes.contiguous()
    index = _check_device("q k_cache v_cache k_len slopes pos k_pos", q, k_cache, v_cache, k_len, slopes, pos, k_pos)
    return _ops.calls().scene_attn_step(_columns(q), _columns(k_cache), _columns(v_cache), k_len.contiguous(), layout.tables(index)[4], layout.max_rows,
                                        slopes, pos, k_pos, scale, softcap)


class RotaryAxes(_Tables):
    """Frequencies of rotary positions with several axes: ``pairs`` = how many column pairs every axis turns (time, y, x, ...; together at most
    head_dim / 2, what is left passes through).  Pair i of an axis of n pairs has the frequency theta ** (-i / n) per unit of the
    axis's position; theta: one number or one per axis.  interleaved: a pair is columns (2 i, 2 i + 1) instead of (i, P + i), P = all
    pairs."""

    def __init__(self, head_dim: int, pairs: Sequence[int], *, theta: Union[float, Sequence[float]] = 10000.0, interleaved: bool = False, device=None):
        super().__init__()
        self.head_dim, self.pairs, self.interleaved = int(head_dim), tuple(int(n) for n in pairs), bool(interleaved)
        self.axes, self.n_pairs = len(self.pairs), sum(self.pairs)
        if self.axes < 1 or min(self.pairs) < 0 or self.n_pairs < 1 or 2 * self.n_pairs > self.head_dim or self.head_dim > 1024:
            raise DagnetHipError(f"pairs {self.pairs}: together 1 .. {self.head_dim // 2} column pairs of a head of {self.head_dim} (at most 1024)")
        th = np.asarray(theta, dtype=np.float64)
        if th.shape not in ((), (self.axes,)):
            raise DagnetHipError(f"theta must be one number or one per axis ({self.axes}), got shape {th.shape}")
        th = np.broadcast_to(th, (self.axes,))
        if not np.all(np.isfinite(th)) or np.any(th <= 0):
            raise DagnetHipError(f"theta must be positive and finite, got {theta}")
        self.freq = np.concatenate([t ** (-np.arange(n, dtype=np.float64) / n) if n else np.zeros(0) for t, n in zip(th, self.pairs)])
        self.axis = np.repeat(np.arange(self.axes, dtype=np.int32), self.pairs)
        if device is not None:
            self.tables(_device(device).index)

    def _host(self):
        turns = self.freq / (2.0 * math.pi)
        return torch.from_numpy(np.concatenate([turns.view(np.uint8), self.axis.view(np.uint8)]))

    def _addresses(self, t):
        return t.data_ptr(), t.data_ptr() + 8 * self.n_pairs                  # turns per unit (fp64), axis


def _apart(a, b) -> bool:
    """No element of the views a and b of one storage is in both, by what their strides show: one lies behind the other, or they share
    strides and their columns differ (a fused projection's q and k, by rows or by heads)."""
    def end(t):
        return t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1

    if not a.numel() or not b.numel() or end(a) <= b.storage_offset() or end(b) <= a.storage_offset():
        return True
    step, cols_a, cols_b = 0, 1, 1                     # elements that repeat every step; what stands in a step
    dims = sorted([(s, n, 0) for s, n in zip(a.stride(), a.shape) if n > 1] + [(s, n, 1) for s, n in zip(b.stride(), b.shape) if n > 1])
    for i, (s, n, which) in enumerate(dims):
        step = 0
        for s2, _, _ in dims[i:]:
            step = math.gcd(step, s2)
        gap = (b.storage_offset() - a.storage_offset()) % step if step else 0
        if step and gap >= cols_a and gap + cols_b <= step:
            return True
        cols_a, cols_b = (cols_a + (n - 1) * s, cols_b) if which == 0 else (cols_a, cols_b + (n - 1) * s)
    return False


def _own_elements(t) -> bool:
    """Every index has an element of its own, by what the strides show."""
    reach = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < reach:
            return False
        reach += (n - 1) * s
    return True


def rotary(q, k, pos, axes: RotaryAxes, *, inplace: bool = False):
    """Turns the column pairs of every head of q [n, heads, head_dim] and k [n, key heads, head_dim] (or None) by their row's positions
    pos [n, number of axes] (fp32, int32 or int64) -> (q, k).  Angles are computed in fp64, so positions may lie far from zero.
    fp32 or bf16, any row and head strides.  Differentiable in q and k; inplace=True overwrites them (without gradient; they must not overlap, and
    autograd sees that they changed)."""
    if not isinstance(axes, RotaryAxes):
        raise DagnetHipError("axes must be RotaryAxes")
    both = (("q", q),) if k is None else (("q", q), ("k", k))
    for name, t in both:
        _matrix3(t, name)
        if t.dtype not in _TYPES or t.dtype != q.dtype:
            raise DagnetHipError(f"q and k must both be fp32 or both bf16 (got {name} {t.dtype})")
        if t.shape[0] != q.shape[0] or t.shape[2] != axes.head_dim or t.shape[1] < 1:
            raise DagnetHipError(f"{name} must be [{q.shape[0]}, heads, {axes.head_dim}], got {tuple(t.shape)}")
    if not isinstance(pos, torch.Tensor) or pos.dtype not in _POSITIONS or tuple(pos.shape) != (q.shape[0], axes.axes):
        raise DagnetHipError(f"pos must be fp32, int32 or int64 [{q.shape[0]}, {axes.axes}]")
    if pos.requires_grad and torch.is_grad_enabled():
        raise DagnetHipError("pos: positions have no gradient here; pass pos.detach()")
    if inplace:
        if torch.is_grad_enabled() and any(t.requires_grad for _, t in both):
            raise DagnetHipError("rotary(inplace=True) has no gradient: call it under torch.no_grad()")
        for name, t in both:
            if t.stride(-1) != 1 and t.shape[-1] > 1 or not _own_elements(t):
                raise DagnetHipError(f"rotary(inplace=True): {name} must have unit column stride and elements of its own (strides {t.stride()})")
        store = [t.untyped_storage().data_ptr() for _, t in both]
        if k is not None and store[0] == store[1] and not _apart(q, k):
            raise DagnetHipError("rotary(inplace=True): q and k overlap")
        if pos.untyped_storage().data_ptr() in store:
            pos = pos.clone()                          # read before anything is overwritten
    tables = axes.tables(_check_device("q k pos", q, k, pos))
    q, k = (q, k) if inplace else (_columns(q), None if k is None else _columns(k))
    return _ops.calls().rotary(q, k, pos.contiguous(), tables, axes.n_pairs, axes.interleaved, inplace)
