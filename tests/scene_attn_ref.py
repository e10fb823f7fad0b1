"""Attention over the rows of a scene in 64 bits, straight from the formulas, with bounds on what a kernel of 32-bit sums may be off by.

x_ij = cap tanh(scale q_i.k_j / cap) - slope_h |pos_i - k_pos_j|, o_i = sum_j softmax_j(x_ij) v_j over the keys j that row i sees.
Everything runs on the CPU, one (row, key) matrix per head.  The bounds follow the arithmetic: u = 2^-24 per fp32 operation, r = 2^-8 per
rounding to bf16 (half a step, relative), a sum of n terms at most n u of the sum of magnitudes."""
import torch

U = 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def seen_matrix(q_ptr, k_ptr=None, causal=0, prefix=0):
    """[nq, nk] truth values from the words of SceneLayout's documentation, row by row."""
    k_ptr = q_ptr if k_ptr is None else k_ptr
    S = len(q_ptr) - 1
    causal = [causal] * S if isinstance(causal, int) else list(causal)
    prefix = [prefix] * S if isinstance(prefix, int) else list(prefix)
    m = torch.zeros((q_ptr[-1], k_ptr[-1]), dtype=torch.bool)
    for s in range(S):
        nq, nk = q_ptr[s + 1] - q_ptr[s], k_ptr[s + 1] - k_ptr[s]
        for i in range(nq):
            for j in range(nk):
                at = i + nk - nq
                g = causal[s]
                m[q_ptr[s] + i, k_ptr[s] + j] = g == 0 or j // g <= at // g or j < prefix[s]      # // rounds down: a row before the first key sees none
    return m


def attention(q, k, v, seen, scale, cap=0.0, slopes=None, pos=None, k_pos=None, dout=None):
    """q [nq, H, D], k, v [nk, KV, D] (any type, any device) -> dict of fp64 results (out; with dout also dq, dk, dv, dslopes), and of the
    bounds of each, for kernels that hold everything in fp32 and round p, ds and the results to the inputs' type."""
    dt = q.dtype
    r = ROUND[dt]
    cpu = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    q, k, v, slopes, pos, k_pos, dout = map(cpu, (q, k, v, slopes, pos, k_pos, dout))
    H, D, KV = q.shape[1], q.shape[2], k.shape[1]
    G = H // KV
    n = seen.sum(1, keepdim=True).double()                       # keys of a row
    m = seen.sum(0, keepdim=True).double().t() * G               # rows of a key
    names = ["out"] + (["dq", "dk", "dv", "dslopes"] if dout is not None else [])
    res = dict(out=torch.zeros_like(q), dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v), dslopes=torch.zeros(H, dtype=torch.float64))
    tol = {a: torch.zeros_like(b) for a, b in res.items()}
    dist = None
    if slopes is not None:
        dist = (pos[:, None, :] - k_pos[None, :, :]).square().sum(-1).sqrt()
    for h in range(H):
        c = h // G
        qh, kh, vh = q[:, h], k[:, c], v[:, c]
        x = qh @ kh.t() * scale
        ex = U * (D + 4) * (qh.abs() @ kh.abs().t()) * abs(scale) + 2 * U * x.abs()
        t = None
        if cap:
            t = torch.tanh(x / cap)
            x = cap * t
            ex = ex + 8 * U * cap * t.abs() + 4 * U * cap          # tanh to a few ulp, its argument's roundings are in the first term
        if dist is not None:
            x = x - slopes[h] * dist
            ex = ex + 8 * U * slopes[h].abs() * dist
        ex = ex + 4 * U * x.abs() + 4 * U
        x = x.masked_fill(~seen, float("-inf"))
        ex = torch.where(seen, ex, torch.zeros_like(ex))
        top = x.amax(1, keepdim=True) if x.shape[1] else x.new_zeros((x.shape[0], 1))
        p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        tot = p.sum(1, keepdim=True)
        p = p / torch.where(tot == 0, torch.ones_like(tot), tot)
        rel = 2 * (ex.amax(1, keepdim=True) if x.shape[1] else 0.0) + (n + 16) * U           # of a probability: its own score and the normaliser's
        o = p @ vh
        eo = (rel + n * U + r) * (p @ vh.abs())                     # r: p rounded for the product
        res["out"][:, h] = o
        tol["out"][:, h] = eo + r * o.abs() + U * o.abs()
        if dout is None:
            continue
        g = dout[:, h]
        dp = g @ vh.t()
        edp = U * (D + 2) * (g.abs() @ vh.abs().t())
        delta = (g * o).sum(1, keepdim=True)
        edelta = (g.abs() * eo).sum(1, keepdim=True) + U * (D + 2) * (g.abs() * o.abs()).sum(1, keepdim=True)
        ds = p * (dp - delta)
        eds = p * (edp + edelta) + (rel + 4 * U) * ds.abs()
        if dist is not None:
            res["dslopes"][h] = -(ds * dist).sum()
            # a row's sums in fp32 over its keys, then fp64 over the rows.  delta's error has no part in it: a row's ds add up to nothing, so
            # what they do add up to is taken back, weighted with the row's mean distance.
            e = p * edp + (rel + (n + 8) * U) * ds.abs()
            mean = (p * dist).sum(1, keepdim=True)
            tol["dslopes"][h] = (e * (dist + mean)).sum() + (edelta * (rel + n * U) * 2 * mean).sum() + U * abs(res["dslopes"][h])
        if cap:
            # (ds + e) (f + d) - ds f = e f + ds d + e d, f = 1 - t^2, d its error.  The last term is what is left in a row with one key, where ds
            # is 0 but for e, under a saturated cap, where f is 0 but for d.
            f, ef = 1 - t * t, 2 * t.abs() * (ex / cap + 12 * U) + 4 * U
            ds, eds = ds * f, eds * f + ds.abs() * ef + eds * ef
        eds = eds + r * ds.abs()
        res["dq"][:, h] = ds @ kh * scale
        tol["dq"][:, h] = (eds @ kh.abs() + n * U * (ds.abs() @ kh.abs())) * abs(scale)
        res["dk"][:, c] += ds.t() @ qh * scale
        tol["dk"][:, c] += (eds.t() @ qh.abs() + m * U * (ds.abs().t() @ qh.abs())) * abs(scale)
        res["dv"][:, c] += p.t() @ g
        tol["dv"][:, c] += (p * (rel + r)).t() @ g.abs() + m * U * (p.t() @ g.abs())
    # A probability below 2^-126 = 1.2e-38 has no normal fp32 value and comes out as 0; what it is multiplied by stays below 10^7 in these
    # tests (sums of |do||v||q|), so a result is off by less than 10^-30 for it.
    for a in names:
        tol[a] = tol[a] + 1e-30
    for a in ("dq", "dk", "dv"):
        tol[a] = tol[a] + (r + 2 * U) * res[a].abs()
    return {a: res[a] for a in names}, {a: tol[a] for a in names}


def close(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want).abs() - tol
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert (over <= 0).all(), f"{what}: off by {float((got - want).abs().max()):.3e}, {float(((got - want).abs() / (tol + 1e-300)).max()):.2f} times the bound"


def turned(x, pos, freq, axis, interleaved, inverse=False):
    """Rotary positions in 64 bits."""
    x = x.detach().cpu().double()
    ang = pos.detach().cpu().double()[:, axis] * torch.as_tensor(freq, dtype=torch.float64)
    P = len(freq)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None] * (-1.0 if inverse else 1.0)
    i = torch.arange(P)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, P + i)
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y
