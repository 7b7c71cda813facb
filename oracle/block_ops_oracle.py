"""Float64 statements of the operators around the layer (test infrastructure, not product code).

``norm_tail``, ``routing`` and ``coefficients`` give each operator's results and gradients in 64 bits, written as formulas, and
next to each result a bound on what 32-bit arithmetic with one final rounding may be off.  A bound is made of

* half a step of the storage type, ``finfo(dtype).eps / 2`` relative to the value, for the final rounding;
* ``U = 2**-24`` times the number of roundings on the longest path to the value, times the sum of the magnitudes of the terms it
  is made of (the same formula evaluated on absolute values).

The path lengths are counted for sums made of at most 64 terms in a row per thread and trees above that; sums over tokens
count every token.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
# longest chain of roundings through one row sum: 32 products per lane, 5 + 16 steps of the tree, sqrt, division
ROW = 64


def half_step(dtype) -> float:
    return 0.0 if dtype == torch.float64 else torch.finfo(dtype).eps / 2


def _sig(g):
    return 1.0 / (1.0 + torch.exp(-g))


def norm_tail(y, residual=None, gate=None, layer_scale=None, post=None, nxt=None, d_out=None, d_normed=None):
    """Values and bounds of ``residual_norm``.  ``post`` / ``nxt`` are ``(weight, eps)``; returns {name: (value, bound)} with the names
    out, normed and, when an upstream gradient is given, y, residual, gate, layer_scale, post, nxt."""
    dt, rt = y.dtype, (y if residual is None else residual).dtype
    f = lambda t: None if t is None else t.double()
    y, res, g, ls = f(y), f(residual), f(gate), f(layer_scale)
    rows, d = y.shape
    one = torch.ones((), dtype=torch.float64)
    rho0 = torch.ones(rows, 1, dtype=torch.float64)
    w0 = one
    if post is not None:
        w0 = f(post[0])
        rho0 = (y.pow(2).sum(-1, keepdim=True) / d + post[1]).rsqrt()
    h = y * rho0
    a = h * w0
    s = one if g is None else g * _sig(g)
    l = one if ls is None else ls
    v = a * s
    r = torch.zeros_like(y) if res is None else res
    out = r + l * v
    mag_out = r.abs() + (l * v).abs()                       # what `out` is the sum of
    # relative error of v: the norm, expf of an argument up to |g| (its relative error grows with it), a few products
    rel_v = (ROW + 16 + (0 if g is None else 2 * g.abs())) * U
    err_out = rel_v * (l * v).abs() + U * mag_out
    got = {"out": (out, half_step(rt) * out.abs() + err_out)}
    rho1 = None
    if nxt is not None:
        w1 = f(nxt[0])
        rho1 = (out.pow(2).sum(-1, keepdim=True) / d + nxt[1]).rsqrt()
        x = out * rho1
        # relative error of rho1: half of the one of mean(out^2)
        rel_rho1 = (out.abs() * err_out).sum(-1, keepdim=True) / d * rho1 ** 2 + ROW * U
        normed = x * w1
        err_x = rho1 * err_out + x.abs() * (rel_rho1 + 4 * U)
        got["normed"] = (normed, half_step(dt) * normed.abs() + w1.abs() * err_x)
    if d_out is None and d_normed is None:
        return got
    dO = torch.zeros_like(y) if d_out is None else d_out.double()
    dR, mag, err = dO, dO.abs(), torch.zeros_like(y)        # err: bound of |dR - computed dR|
    if d_normed is not None:
        dN = d_normed.double()
        u = w1 * dN
        m = (u * x).mean(-1, keepdim=True)
        dR = dO + rho1 * (u - x * m)
        mag_m = (u * x).abs().mean(-1, keepdim=True)
        err_m = (u.abs() * err_x).mean(-1, keepdim=True) + ROW * U * mag_m
        mag = dO.abs() + rho1 * (u.abs() + x.abs() * mag_m)
        err = rho1 * (err_x * m.abs() + x.abs() * err_m) + (rel_rho1 + 8 * U) * rho1 * (u.abs() + x.abs() * mag_m) + 2 * U * mag
    got["residual"] = (dR, half_step(rt) * dR.abs() + err)
    n_sum = (rows + 128) * U
    if ls is not None:
        dls = (dR * v).sum(0)
        got["layer_scale"] = (dls, half_step(dt) * dls.abs() + (err * v.abs() + rel_v * (dR * v).abs()).sum(0) + n_sum * (mag * v.abs()).sum(0))
    dv, err_dv = l * dR, l.abs() * err + U * (l * dR).abs()
    if g is not None:
        sg = _sig(g)
        ds = sg * (1.0 + g * (1.0 - sg))
        mag_ds = sg * (1.0 + g.abs() * (1.0 - sg))
        dg = dv * a * ds
        rel_ds = (16 + 4 * g.abs()) * U
        got["gate"] = (dg, half_step(dt) * dg.abs() + err_dv * (a * ds).abs() + (dv * a).abs() * (rel_ds * mag_ds + ROW * U * ds.abs()))
    da = dv * s
    err_da = err_dv * s.abs() + (16 + (0 if g is None else 2 * g.abs())) * U * da.abs()
    if post is None:
        got["y"] = (da, half_step(dt) * da.abs() + err_da)
    else:
        b = (w0 * da * h)
        m0 = b.mean(-1, keepdim=True)
        # m0 comes from three sums: sum q*b, and mean(u*x) * rho1 * sum q*x; their magnitudes are what rounds
        q = w0 * l * s * h
        mag_b = dO.abs() + (0 if d_normed is None else (rho1 * u).abs())
        mag_m0 = (q.abs() * mag_b).mean(-1, keepdim=True)
        if d_normed is not None:
            mag_m0 = mag_m0 + rho1 * mag_m * (q * x).abs().mean(-1, keepdim=True)
        err_m0 = (w0.abs() * err_da * h.abs()).mean(-1, keepdim=True) + 3 * (ROW + 32 + (0 if g is None else 2 * g.abs().amax(-1, keepdim=True))) * U * mag_m0
        dy = rho0 * (w0 * da - h * m0)
        mag_dy = rho0 * ((w0 * da).abs() + h.abs() * mag_m0)
        got["y"] = (dy, half_step(dt) * dy.abs() + rho0 * (w0.abs() * err_da + h.abs() * err_m0) + 2 * ROW * U * mag_dy)
        dw0 = (da * h).sum(0)
        got["post"] = (dw0, half_step(dt) * dw0.abs() + (err_da * h.abs() + ROW * U * (da * h).abs()).sum(0) + n_sum * (da * h).abs().sum(0))
    if nxt is not None:
        if d_normed is None:
            got["nxt"] = (torch.zeros(d, dtype=torch.float64), torch.zeros(d, dtype=torch.float64))
        else:
            dw1 = (dN * x).sum(0)
            got["nxt"] = (dw1, half_step(dt) * dw1.abs() + (dN.abs() * err_x).sum(0) + n_sum * (dN * x).abs().sum(0))
    return got


def routing(scores, top_k, mask=None, router=(0, 10.0, 0.5), d_gates=None, d_balance=None, d_z=None):
    """Values and bounds of ``route_tokens``: idx and counts (exact), and (value, bound) for gates, balance, z and scores (the
    gradient, when an upstream gradient is given).  ``scores`` (T, E) without NaN in tokens that count."""
    dt = scores.dtype
    x = scores.double()
    T, E = x.shape
    rule, cap, temp = router
    on = ~torch.isneginf(x)
    live = on.any(-1) if mask is None else (on.any(-1) & mask)
    on = on & live[:, None]
    x = torch.where(on, x, torch.full_like(x, -torch.inf))   # a token that does not count has no experts
    idx = torch.full((T, top_k), -1, dtype=torch.int32)
    for t in range(T):
        order = sorted((e for e in range(E) if on[t, e]), key=lambda e: (-float(x[t, e]), e))[:top_k]
        idx[t, :len(order)] = torch.tensor(order, dtype=torch.int32)
    counts = torch.stack([(idx == e).sum() for e in range(E)]).to(torch.int32)
    arg = torch.where(on, x, torch.zeros_like(x)) / cap
    l = torch.where(on, cap * torch.tanh(arg) / temp if rule else x, torch.full_like(x, -torch.inf))
    top = torch.where(live, l.amax(-1), torch.zeros(T, dtype=torch.float64))[:, None]
    ex = torch.where(on, torch.exp(l - top), torch.zeros_like(l))
    den = torch.where(live[:, None], ex.sum(-1, keepdim=True), torch.ones(T, 1, dtype=torch.float64))
    p = ex / den
    lse = torch.where(live, (top + torch.log(den))[:, 0], torch.zeros(T, dtype=torch.float64))
    # error of a logit: rule 1 makes it with a division, a tanh of 2 ulp, two products; then the difference to the largest, expf
    big = torch.where(on, l.abs(), torch.zeros_like(l)).amax(-1, keepdim=True)
    err_l = (16 * big if rule else 2 * big) * U
    rel_p = 2 * err_l + (ROW + 8) * U + 2 * big * U
    n = int(live.sum())
    sel = idx.clamp(min=0).long()
    full = idx >= 0
    won = torch.where(full, ex.gather(1, sel), torch.zeros(T, top_k, dtype=torch.float64))
    if rule:
        pw = won / den
        gates = pw / (pw.sum(-1, keepdim=True) + 1e-6)
    else:
        gates = won / torch.where(live[:, None], won.sum(-1, keepdim=True), torch.ones(T, 1, dtype=torch.float64))
    inv = 1.0 / n if n else 0.0
    fr = counts.double() * inv / top_k
    P = p.sum(0) * inv
    balance = E * (fr * P).sum()
    z = lse.pow(2).sum() * inv
    chain = (T + 512) * U
    rel_mean = rel_p.amax() if T else 0.0
    err_lse = err_l[:, 0] + (ROW + 8) * U + 2 * lse.abs() * U
    got = {"idx": idx, "counts": counts, "gates": (gates, 3 * rel_p * gates),
           "balance": (balance, (rel_mean + chain) * balance),
           "z": (z, (2 * lse.abs() * err_lse).sum() * inv + (chain + 4 * U) * z)}
    if d_gates is None and d_balance is None and d_z is None:
        return got
    A = (0.0 if d_balance is None else float(d_balance)) * E * fr * inv
    c_z = (0.0 if d_z is None else float(d_z)) * 2.0 * inv * lse[:, None]
    pA = (p * A).sum(-1, keepdim=True)
    dl = p * (A - pA + c_z)
    mag = p * (A.abs() + (p * A.abs()).sum(-1, keepdim=True) + c_z.abs())
    err = p * abs(0.0 if d_z is None else float(d_z)) * 2.0 * inv * err_lse[:, None]
    if d_gates is not None:
        dg = torch.where(full, d_gates.double(), torch.zeros(T, top_k, dtype=torch.float64))
        G = (gates * dg).sum(-1, keepdim=True)
        mag_G = (gates * dg.abs()).sum(-1, keepdim=True)
        dl = dl.scatter_add(1, sel, torch.where(full, gates * (dg - G), torch.zeros_like(gates)))
        mag = mag.scatter_add(1, sel, torch.where(full, gates * (dg.abs() + mag_G), torch.zeros_like(gates)))
        if rule:
            rest = 1.0 - gates.sum(-1, keepdim=True)
            dl = dl - p * G * rest
            mag = mag + p * mag_G * (rest.abs() + 1.0)     # 1 - sum of gates cancels
    ds = torch.ones_like(x)
    rel_ds = 0.0
    if rule:
        ds = torch.cosh(arg).pow(-2) / temp
        rel_ds = (16 + 4 * arg.abs()) * U
    val = torch.where(on, dl * ds, torch.zeros_like(dl))
    bound = half_step(dt) * val.abs() + ds * (mag * (6 * rel_p + 2 * ROW * U + rel_ds) + err)
    got["scores"] = (val, torch.where(on, bound, torch.zeros_like(bound)))
    return got


def coefficients(idx, gates, u, d_c=None):
    """Values and bounds of ``expert_coefficients``: {c, gates, u: (value, bound)}; idx (T, k)."""
    T, k = idx.shape
    E, r1 = u.shape
    g, w = gates.double(), u.double()
    c = torch.zeros(T, r1, dtype=torch.float64)
    mag = torch.zeros_like(c)
    d_g, mag_g = torch.zeros(T, k, dtype=torch.float64), torch.zeros(T, k, dtype=torch.float64)
    d_u, mag_u = torch.zeros(E, r1, dtype=torch.float64), torch.zeros(E, r1, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = int(idx[t, j])
            if not 0 <= e < E:
                continue
            c[t] += g[t, j] * w[e]
            mag[t] += (g[t, j] * w[e]).abs()
            if d_c is not None:
                dc = d_c[t].double()
                d_g[t, j] = (w[e] * dc).sum()
                mag_g[t, j] = (w[e] * dc).abs().sum()
                d_u[e] += g[t, j] * dc
                mag_u[e] += (g[t, j] * dc).abs()
    got = {"c": (c, (k + 2) * U * mag)}
    if d_c is not None:
        got["gates"] = (d_g, (r1 + 2) * U * mag_g)
        got["u"] = (d_u, half_step(u.dtype) * d_u.abs() + (T * k + 256) * U * mag_u)
    return got
