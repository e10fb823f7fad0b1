"""What is measured of the scene-attention operators: attention over the rows of a scene (forward and training), the same for the new
rows of a step over kept keys, and rotary positions with several axes.

`own` False computes each in its plain form (elementary torch operations in 32 bits); True calls the framework."""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attn(name, *, scenes, agents, steps, heads, kv, dim, dtype, train, mask="none", obs=0, cap=0.0, axes=0):
    return {"name": name, "op": "attn", "scenes": scenes, "agents_lo": agents[0], "agents_hi": agents[1], "steps_lo": steps[0],
            "steps_hi": steps[1], "heads": heads, "kv": kv, "dim": dim, "dtype": dtype, "train": train, "mask": mask, "obs": obs,
            "cap": cap, "axes": axes}


def _step(name, *, scenes, agents, steps, room, heads, kv, dim, dtype, cap=0.0, axes=0):
    return {"name": name, "op": "step", "scenes": scenes, "agents_lo": agents[0], "agents_hi": agents[1], "steps_lo": steps[0],
            "steps_hi": steps[1], "room": room, "heads": heads, "kv": kv, "dim": dim, "dtype": dtype, "cap": cap, "axes": axes}


def _rotary(name, *, rows, heads, kv, dim, pairs, dtype, train, interleaved, far):
    return {"name": name, "op": "rotary", "rows": rows, "heads": heads, "kv": kv, "dim": dim, "pairs": pairs, "dtype": dtype,
            "train": train, "interleaved": interleaved, "far": far}


def listed():
    return [
        # one basketball scene: the ten players of one time step look at each other, weighted by their distance (latency)
        _attn("one_scene", scenes=1, agents=(10, 10), steps=(1, 1), heads=4, kv=4, dim=16, dtype="fp32", train=False, axes=2),
        # the graph layer of a basketball training batch: 4096 scenes of ten players
        _attn("players_train", scenes=4096, agents=(10, 10), steps=(1, 1), heads=4, kv=4, dim=16, dtype="fp32", train=True, axes=2),
        # the same for drone footage: 1 to 32 people in a scene
        _attn("crowd_train", scenes=1024, agents=(1, 32), steps=(1, 1), heads=4, kv=4, dim=40, dtype="fp32", train=True, axes=2),
        # whole basketball sequences, ten players by fifty steps: the ten observed steps are a prefix that all rows see, later ones are
        # causal by time step; capped scores and a decay with the distance in time and on the court
        _attn("sequence_train", scenes=32, agents=(10, 10), steps=(50, 50), heads=8, kv=8, dim=64, dtype="bf16", train=True,
              mask="prefix", obs=10, cap=30.0, axes=3),
        # whole drone sequences (8 observed and 12 further steps), ragged, keys and values shared by two heads each
        _attn("crowd_sequence_train", scenes=48, agents=(3, 17), steps=(20, 20), heads=4, kv=2, dim=32, dtype="fp32", train=True,
              mask="prefix", obs=8, axes=2),
        # long recordings as one causal sequence each, forward
        _attn("long_forward", scenes=2, agents=(1, 1), steps=(6145, 8192), heads=16, kv=4, dim=128, dtype="bf16", train=False,
              mask="causal", cap=50.0, axes=1),
        # a long recording of odd length and head width, training
        _attn("long_train", scenes=1, agents=(1, 1), steps=(4093, 4093), heads=8, kv=2, dim=96, dtype="bf16", train=True, mask="causal"),
        # a rollout's step of one scene over its fifty kept steps (latency)
        _step("step_one_scene", scenes=1, agents=(10, 10), steps=(50, 50), room=500, heads=4, kv=4, dim=16, dtype="fp32", axes=2),
        # a step of many scenes, ten rows each, over up to two hundred kept steps
        _step("step_batch", scenes=256, agents=(7, 10), steps=(40, 200), room=2000, heads=8, kv=2, dim=64, dtype="bf16", cap=30.0, axes=3),
        # one row a sequence over very long kept sequences
        _step("step_long", scenes=4, agents=(1, 1), steps=(60000, 131071), room=131072, heads=16, kv=4, dim=128, dtype="bf16"),
        # positions of a rollout's step
        _rotary("rotary_step", rows=10, heads=8, kv=2, dim=64, pairs="12,10,10", dtype="bf16", train=False, interleaved=False, far=200.0),
        # positions of a training batch of long recordings (time stamps far from zero), with the gradients
        _rotary("rotary_train", rows=65521, heads=16, kv=4, dim=128, pairs="32,16,16", dtype="bf16", train=True, interleaved=False, far=1e6),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the ranges above: scenes of one to 32 agents, one time step to long sequences, every type and mask."""
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("attn", "attn", "step", "rotary"))
        kv = rng.choice((1, 2, 3, 4, 8))
        heads = kv * rng.choice((1, 1, 2, 3, 4))
        dim = rng.choice((8, 16, 20, 32, 40, 48, 64, 72, 80, 96, 100, 128))
        dtype = rng.choice(("fp32", "bf16"))
        cap = rng.choice((0.0, 0.0, 20.0, 50.0))
        axes = rng.choice((0, 1, 2, 3))
        lo = _log(rng, 1, 16)
        agents = (lo, _log(rng, lo, 32))
        if op == "attn":
            shape = rng.choice(("agents", "sequence", "long"))
            train = rng.random() < 0.6
            if shape == "agents":
                c = _attn("", scenes=_log(rng, 1, 4096), agents=agents, steps=(1, 1), heads=heads, kv=kv, dim=dim, dtype=dtype, train=train,
                          cap=cap, axes=axes)
            elif shape == "sequence":
                t = _log(rng, 5, 60)
                c = _attn("", scenes=_log(rng, 1, 48), agents=agents, steps=(max(2, t // 2), t), heads=heads, kv=kv, dim=dim, dtype=dtype,
                          train=train, mask=rng.choice(("none", "causal", "prefix")), obs=rng.randint(1, 8), cap=cap, axes=axes)
            else:
                t = _log(rng, 500, 4096)
                c = _attn("", scenes=_log(rng, 1, 4), agents=(1, 1), steps=(rng.randint(t // 2, t), t), heads=heads, kv=kv, dim=dim,
                          dtype=dtype, train=train, mask=rng.choice(("causal", "prefix", "none")), obs=rng.randint(1, 200), cap=cap, axes=axes)
        elif op == "step":
            scenes = _log(rng, 1, 256)
            t = _log(rng, 16, 131072)
            if scenes * t * agents[1] > 600000:
                continue
            c = _step("", scenes=scenes, agents=agents, steps=(rng.randint(max(1, t // 2), t), t), room=t * agents[1] + rng.randint(0, 50),
                      heads=heads, kv=kv, dim=dim, dtype=dtype, cap=cap, axes=axes)
        else:
            dim = rng.choice((16, 32, 48, 64, 80, 96, 128))
            n = dim // 2
            a = rng.randint(1, n - 2)
            b = rng.randint(1, n - a - 1)
            pairs = rng.choice(("%d" % n, "%d,%d" % (a, n - a), "%d,%d,%d" % (a, b, n - a - b)))
            c = _rotary("", rows=_log(rng, 1, 65536), heads=heads, kv=kv, dim=dim, pairs=pairs, dtype=dtype, train=rng.random() < 0.5,
                        interleaved=rng.random() < 0.5, far=float(_log(rng, 10, 1000000)))
        if _cost(c) <= top:
            del c["name"]
            return c


def _cost(case):
    w = work(case)
    return w["flops"] + 100.0 * w["bytes"]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _scenes(case):
    """Agents and time steps of every scene: part of the case, like a data set's scene lengths."""
    r = random.Random(",".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))
    n = case["scenes"]
    return ([r.randint(case["agents_lo"], case["agents_hi"]) for _ in range(n)], [r.randint(case["steps_lo"], case["steps_hi"]) for _ in range(n)])


def _pairs_seen(a, t, mask, obs):
    """Pairs (row, visible key) of a scene of `a` agents by `t` steps."""
    if mask == "none":
        return (a * t) ** 2
    p = min(obs, t) if mask == "prefix" else 0
    return a * a * sum(max(i + 1, p) for i in range(t)) if t <= 64 else a * a * (p * p + (t * (t + 1) - p * (p + 1)) // 2)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    H, KV, D = case["heads"], case["kv"], case["dim"]
    if case["op"] == "rotary":
        x = case["rows"] * (H + KV) * D
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * x * size + case["rows"] * 4 * len(case["pairs"].split(",")), "flops": passes * 3 * x}
    agents, steps = _scenes(case)
    if case["op"] == "step":
        rows, keys = sum(agents), [a * t for a, t in zip(agents, steps)]
        pairs = sum(a * k for a, k in zip(agents, keys))
        return {"bytes": size * (2 * rows * H * D + 2 * sum(keys) * KV * D) + 4 * case["axes"] * (rows + sum(keys)), "flops": 4 * D * H * pairs}
    rows = sum(a * t for a, t in zip(agents, steps))
    pairs = sum(_pairs_seen(a, t, case["mask"], case["obs"]) for a, t in zip(agents, steps))
    bytes_ = size * rows * D * (2 * H + 2 * KV) + 4 * case["axes"] * rows
    if case["train"]:
        bytes_ += size * rows * D * (2 * H + 2 * KV)       # the gradient of the output read, those of the inputs written
        return {"bytes": bytes_, "flops": 14 * D * H * pairs}
    return {"bytes": bytes_, "flops": 4 * D * H * pairs}


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _walk(gen, rows, agent, step, axes):
    """Positions of the rows: the time step, then y and x on a court of 50 by 94 feet."""
    xy = torch.rand((rows, 2), generator=gen, device=DEV) * torch.tensor([50.0, 94.0], device=DEV)
    p = torch.cat([step[:, None].float(), xy], 1)
    return None if axes == 0 else {1: p[:, :1], 2: p[:, 1:], 3: p}[axes].contiguous()


def _slopes(heads):
    """Decay per unit of distance: a geometric row, the usual choice."""
    return torch.tensor([2.0 ** (-1.0 - 6.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device=DEV)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 1000003 + 17)
    dt = TYPES[case["dtype"]]
    H, KV, D = case["heads"], case["kv"], case["dim"]
    if case["op"] == "rotary":
        N, pairs = case["rows"], [int(v) for v in case["pairs"].split(",")]
        s = {"q": _normal(gen, (N, H, D), dt), "k": _normal(gen, (N, KV, D), dt),
             "pos": torch.rand((N, len(pairs)), generator=gen, device=DEV) * case["far"], "pairs": pairs}
        s["pos"][:, 0] = s["pos"][:, 0].floor()
        if case["train"]:
            s["dq"], s["dk"] = _normal(gen, (N, H, D), dt), _normal(gen, (N, KV, D), dt)
        return s
    agents, steps = _scenes(case)
    S = len(agents)
    rows = agents if case["op"] == "step" else [a * t for a, t in zip(agents, steps)]
    ptr = np.concatenate([[0], np.cumsum(rows)]).astype(np.int64)
    N = int(ptr[-1])
    scene = np.repeat(np.arange(S), rows)
    local = np.arange(N) - ptr[scene]
    agent_n = np.asarray(agents)[scene]
    s = {"ptr": ptr, "agents": agents, "steps": steps, "most": max(rows), "scale": 1.0 / math.sqrt(D)}
    to = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(DEV)  # noqa: E731
    # scenes side by side with room for the longest: where each row stands there, and which row stands at each place
    s["at"] = to(scene * s["most"] + local)
    inside = np.arange(s["most"])[None, :] < np.asarray(rows)[:, None]
    spare = (np.arange(S * s["most"]) % N).reshape(S, s["most"])            # what stands in the room left over is not looked at
    s["rows"] = to(np.where(inside, ptr[:-1, None] + np.arange(s["most"])[None, :], spare))
    s["n"] = to(np.asarray(rows))
    s["agents_dev"] = to(np.asarray(agents))
    # scores of a trained layer: a few keys stand out
    s["q"] = _normal(gen, (N, H, D), dt, 1.5)
    s["slopes"] = _slopes(H) if case["axes"] else None
    if case["op"] == "step":
        C = case["room"]
        s["k"], s["v"] = _normal(gen, (S, C, KV, D), dt), _normal(gen, (S, C, KV, D), dt)
        s["k_len"] = to(np.asarray([a * t for a, t in zip(agents, steps)], dtype=np.int32))
        when = to(np.broadcast_to(np.arange(C)[None, :], (S, C)).reshape(-1)) // s["agents_dev"].repeat_interleave(C)
        kp = _walk(gen, S * C, None, when, case["axes"])
        s["k_pos"] = None if kp is None else kp.view(S, C, -1)
        s["pos"] = _walk(gen, N, None, to(np.asarray(steps)[scene] - 1), case["axes"])
        return s
    s["k"], s["v"] = _normal(gen, (N, KV, D), dt), _normal(gen, (N, KV, D), dt)
    s["pos"] = _walk(gen, N, None, to(local // agent_n), case["axes"])
    if case["train"]:
        s["dout"] = _normal(gen, (N, H, D), dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "rotary":
        freq, axis = _frequencies(s["pairs"])
        s["freq"], s["axis"] = torch.tensor(freq, dtype=torch.float64, device=DEV), torch.tensor(axis, device=DEV)
    if case.get("train"):
        s["leaves"] = [s[n].requires_grad_() for n in (("q", "k") if case["op"] == "rotary" else ("q", "k", "v"))]
        if s.get("slopes") is not None:
            s["leaves"].append(s["slopes"].requires_grad_())
    if own:                                  # the handles that a program makes once for its batch layout and its head width
        from dagnet_amd.attention import RotaryAxes, SceneLayout
        if case["op"] == "rotary":
            s["axes"] = RotaryAxes(case["dim"], s["pairs"], interleaved=case["interleaved"], device=DEV)
        elif case["op"] == "step":
            s["layout"] = SceneLayout(s["ptr"], device=DEV)
        else:
            groups, prefix = s["agents"], [a * case["obs"] for a in s["agents"]]
            s["layout"] = SceneLayout(s["ptr"], causal=groups if case["mask"] != "none" else 0,
                                      prefix=prefix if case["mask"] == "prefix" else 0, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _frequencies(pairs, theta=10000.0):
    """Frequency and axis of every pair: theta ** (-i / n) for pair i of an axis of n pairs."""
    return [theta ** (-i / n) for n in pairs for i in range(n)], [a for a, n in enumerate(pairs) for _ in range(n)]


def _distance(a, b):
    """[S, n, A], [S, m, A] -> [S, n, m]"""
    return (a[:, :, None, :] - b[:, None, :, :]).square().sum(-1).sqrt()


def _visible(case, s):
    """[S, rows, keys] truth values."""
    n, most, dev = s["n"], s["most"], s["q"].device
    if case["op"] == "step":
        keys = s["k"].shape[1]
        return (torch.arange(keys, device=dev)[None, None, :] < s["k_len"][:, None, None]).expand(-1, most, -1)
    i = torch.arange(most, device=dev)
    seen = (i[None, None, :] < n[:, None, None]).expand(-1, most, -1)
    if case["mask"] == "none":
        return seen
    a = s["agents_dev"][:, None]
    end = (i[None, :] // a + 1) * a
    if case["mask"] == "prefix":
        end = torch.maximum(end, a * case["obs"])
    return seen & (i[None, None, :] < end[:, :, None])


def _plain_attention(case, s, q, k, v, slopes):
    S, H, KV, D = len(s["agents"]), case["heads"], case["kv"], case["dim"]
    side = lambda x: x.float()[s["rows"]]  # noqa: E731  packed rows -> [S, most, ..]
    qs = side(q).view(S, s["most"], KV, H // KV, D).permute(0, 2, 3, 1, 4)
    ks, vs = (k.float(), v.float()) if case["op"] == "step" else (side(k), side(v))
    ks, vs = ks.permute(0, 2, 3, 1)[:, :, None], vs.permute(0, 2, 1, 3)[:, :, None]
    x = torch.matmul(qs, ks) * s["scale"]
    if case["cap"]:
        x = torch.tanh(x / case["cap"]) * case["cap"]
    if case["axes"]:
        pos = side(s["pos"])
        x = x - slopes.view(1, KV, H // KV, 1, 1) * _distance(pos, s["k_pos"] if case["op"] == "step" else pos)[:, None, None]
    x = x.masked_fill(~_visible(case, s)[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True).detach()
    p = torch.exp(x - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, vs) / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 3, 1, 2, 4).reshape(S * s["most"], H, D)[s["at"]].to(q.dtype)


def _plain_turn(x, cos, sin, interleaved):
    P = cos.shape[-1]
    y = x.float()
    if interleaved:
        a, b = y[..., 0:2 * P:2], y[..., 1:2 * P:2]
        t = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :P], y[..., P:2 * P]
        t = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([t, y[..., 2 * P:]], -1).to(x.dtype)


def _plain_rotary(case, s, q, k):
    angle = s["pos"].double()[:, s["axis"]] * s["freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    return _plain_turn(q, cos, sin, case["interleaved"]), _plain_turn(k, cos, sin, case["interleaved"])


def _forward(case, s):
    if case["op"] == "rotary":
        if own:
            from dagnet_amd.attention import rotary
            return rotary(s["q"], s["k"], s["pos"], s["axes"])
        return _plain_rotary(case, s, s["q"], s["k"])
    if not own:
        return (_plain_attention(case, s, s["q"], s["k"], s["v"], s["slopes"]),)
    from dagnet_amd.attention import scene_attention, scene_attention_step
    if case["op"] == "step":
        return (scene_attention_step(s["q"], s["k"], s["v"], s["k_len"], s["layout"], softcap=case["cap"], slopes=s["slopes"],
                                     pos=s["pos"], k_pos=s["k_pos"]),)
    return (scene_attention(s["q"], s["k"], s["v"], s["layout"], softcap=case["cap"], slopes=s["slopes"], pos=s["pos"]),)


def run(state):
    case = state["case"]
    if not case.get("train"):
        with torch.no_grad():
            return _forward(case, state)
    outs = _forward(case, state)
    up = (state["dq"], state["dk"]) if case["op"] == "rotary" else (state["dout"],)
    grads = torch.autograd.grad(outs, state["leaves"], up)
    return [o.detach() for o in outs] + list(grads)


# ---------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_rotary(case, s):
    freq, axis = _frequencies(s["pairs"])
    ang = s["pos"].double()[:, axis] * torch.tensor(freq, dtype=torch.float64, device=DEV)
    P = len(freq)
    first = torch.arange(P, device=DEV) * 2 if case["interleaved"] else torch.arange(P, device=DEV)
    second = first + 1 if case["interleaved"] else first + P

    def turn(x, sign):
        x = x.detach().double()
        y = x.clone()
        c, n = torch.cos(ang)[:, None], torch.sin(ang)[:, None] * sign
        y[..., first] = x[..., first] * c - x[..., second] * n
        y[..., second] = x[..., first] * n + x[..., second] * c
        return y
    out = [turn(s["q"], 1.0), turn(s["k"], 1.0)]
    return out + [turn(s["dq"], -1.0), turn(s["dk"], -1.0)] if case["train"] else tuple(out)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    H, KV, D, cap = case["heads"], case["kv"], case["dim"], case["cap"]
    G, train, ptr = H // KV, case.get("train", False), s["ptr"]
    step = case["op"] == "step"
    pick = lambda x: None if x is None else x.detach().double()  # noqa: E731
    q, pos, slopes, do = pick(s["q"]), pick(s["pos"]), pick(s["slopes"]), pick(s.get("dout"))
    k, v = (s["k"], s["v"]) if step else (pick(s["k"]), pick(s["v"]))
    out = torch.zeros_like(q)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v)) if train else (None,) * 3
    dsl = torch.zeros(H, dtype=torch.float64, device=DEV)
    for i in range(case["scenes"]):
        r = slice(int(ptr[i]), int(ptr[i + 1]))
        a = s["agents"][i]
        m = a * s["steps"][i] if step else r.stop - r.start
        ki, vi = (k[i, :m].double(), v[i, :m].double()) if step else (k[r], v[r])
        dist = None
        if case["axes"]:
            kp = s["k_pos"][i, :m].double() if step else pos[r]
            dist = torch.zeros((r.stop - r.start, m), dtype=torch.float64, device=DEV)
            for c in range(case["axes"]):
                dist += (pos[r][:, c, None] - kp[None, :, c]) ** 2
            dist = dist ** 0.5
        hide = None
        if not step and case["mask"] != "none":
            j = torch.arange(m, device=DEV)
            end = (j // a + 1) * a
            if case["mask"] == "prefix":
                end = end.clamp(min=a * case["obs"])
            hide = j[None, :] >= end[:, None]
        # small scenes take all heads at once, large ones a few at a time
        per = max(1, min(G, int(2 ** 28 // max(1, (r.stop - r.start) * m))))
        for g in range(KV):
            for h0 in range(g * G, (g + 1) * G, per):
                hs = slice(h0, min(h0 + per, (g + 1) * G))
                qh = q[r, hs].transpose(0, 1)
                z = (qh @ ki[:, g].t()) / math.sqrt(D)
                th = None
                if cap:
                    th = torch.tanh(z / cap)
                    z = cap * th
                if dist is not None:
                    z = z - slopes[hs, None, None] * dist
                if hide is not None:
                    z = z.masked_fill(hide, -math.inf)
                p = torch.softmax(z, -1)
                del z
                out[r, hs] = (p @ vi[:, g]).transpose(0, 1)
                if not train:
                    continue
                doh = do[r, hs].transpose(0, 1)
                dp = doh @ vi[:, g].t()
                dz = p * (dp - (p * dp).sum(-1, keepdim=True))
                dv[r, g] += (p.transpose(1, 2) @ doh).sum(0)
                if dist is not None:
                    dsl[hs] -= (dz * dist).sum((1, 2))
                if cap:
                    dz = dz * (1 - th * th)
                dq[r, hs] = ((dz @ ki[:, g]) / math.sqrt(D)).transpose(0, 1)
                dk[r, g] += (dz.transpose(1, 2) @ qh).sum(0) / math.sqrt(D)
    if not train:
        return (out,)
    return [out, dq, dk, dv] + ([dsl] if case["axes"] else [])
