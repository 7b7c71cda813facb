"""Operators around a Tucker-MoE layer, as cases that can be timed and compared.

Three operators of one block, forward alone (serving) or with their gradients (training):

* ``residual_norm``: the tail of a block in one pass over its rows,
  ``out = residual + layer_scale * silu(gate) * norm(y, post_norm)`` and ``normed = norm(out, next_norm)``;
* ``route_tokens``: top-k selection and gate weights from router scores, tokens per expert, the balance loss and the
  z loss;
* ``expert_coefficients``: the coefficient vector ``c[t] = sum_j gates[t, j] * U_expert[idx[t, j]]`` that mixes the
  layer's core slices.

``run`` computes them in plain torch (``own`` false) or through ``mamba_tuckermoe_b200`` (``own`` true); ``exact`` states
them once more in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-5
CAP, TEMPERATURE = 10.0, 0.5          # gate rule 1: soft cap of the scores, softmax temperature
BALANCE_WEIGHT, Z_WEIGHT = 1e-2, 1e-3  # what a training loss multiplies the two router losses by
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- cases
def _norm(name, rows, d, dtype, train, residual="same", scale=True, gate=False, post=False, nxt=True):
    c = {"op": "norm", "rows": rows, "d": d, "dtype": dtype, "train": train, "residual": residual, "scale": scale, "gate": gate,
         "post": post, "next": nxt}
    return dict(c, name=name) if name else c


def _route(name, tokens, experts, k, dtype, train, rule, padded=False, disabled=0):
    c = {"op": "route", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "train": train, "rule": rule, "padded": padded,
         "disabled": disabled}
    return dict(c, name=name) if name else c


def _coef(name, tokens, experts, k, r1, dtype, train, skew):
    c = {"op": "coef", "tokens": tokens, "experts": experts, "k": k, "r1": r1, "dtype": dtype, "train": train, "skew": skew}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token: a block's output added to the residual stream and normed for the next block
        _norm("norm_decode_1", 1, 768, "bf16", False),
        # prefill of a block that norms its output and multiplies it by the gate half of a wider projection
        _norm("norm_prefill_gated", 32768, 768, "bf16", False, gate=True, post=True),
        # odd width in fp32 (no row starts on a 16-byte boundary), no layer scale, with gradients
        _norm("norm_odd_fp32", 777, 1001, "fp32", True, scale=False, gate=True, post=True),
        # training step at a layer's output width: norms before and after, all parameter gradients
        _norm("norm_train", 16384, 2304, "bf16", True, post=True),
        # training with the residual stream kept in fp32 beside bf16 blocks
        _norm("norm_train_fp32_residual", 8192, 1536, "bf16", True, residual="fp32", gate=True),
        # one decode step of a batch of 64 sequences: 8 experts, top-2
        _route("route_decode_64", 64, 8, 2, "bf16", False, 0),
        # a training batch padded at its ends, 64 experts top-2
        _route("route_train_padded", 32768, 64, 2, "bf16", True, 0, padded=True),
        # a ragged batch under the capped rule in fp32, an odd number of experts, some of them switched off
        _route("route_ragged_capped", 4097, 100, 3, "fp32", True, 1, disabled=7),
        # the largest batch: 256 experts, top-8, capped rule, skewed scores
        _route("route_train_large", 131072, 256, 8, "bf16", True, 1),
        # coefficients of one decode step
        _coef("coef_decode_64", 64, 8, 2, 32, "bf16", False, False),
        # coefficients and their gradients for a training batch
        _coef("coef_train", 32768, 64, 2, 4, "bf16", True, False),
        # the same where few experts take most tokens
        _coef("coef_train_skewed", 131072, 256, 8, 8, "bf16", True, True),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is uniform over lo .. hi."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "norm", "route", "route", "coef"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    train = rng.random() < 0.6
    if op == "norm":
        d = _spread(rng, 64, 8192)
        if rng.random() < 0.7:
            d = max(64, d // 8 * 8)
        rows = _spread(rng, 1, max(1, min(131072, (16384 * 2304 // (2 if dtype == "fp32" else 1)) // d)))
        residual = rng.choice(("same", "same", "fp32", "none"))
        scale, gate, post = rng.random() < 0.7, rng.random() < 0.4, rng.random() < 0.5
        nxt = rng.random() < 0.8 or not (residual != "none" or scale or gate or post)
        return _norm(None, rows, d, dtype, train, residual, scale, gate, post, nxt)
    experts = _spread(rng, 2, 1024)
    if rng.random() < 0.5:
        experts = 2 ** int(round(math.log2(experts)))
    k = min(experts, rng.choice((1, 2, 2, 3, 4, 6, 8, 8)))
    if op == "route":
        tokens = _spread(rng, 1, min(131072, 131072 * 256 // (2 if dtype == "fp32" else 1) // experts))
        disabled = rng.randrange(0, experts // 4 + 1) if rng.random() < 0.3 else 0
        return _route(None, tokens, experts, k, dtype, train, rng.randrange(2), rng.random() < 0.5, disabled)
    r1 = rng.choice((2, 3, 4, 7, 8, 16, 32, 32, 64))
    tokens = _spread(rng, 1, min(131072, 131072 * 8 * 8 // (k * r1)))
    return _coef(None, tokens, experts, k, r1, dtype, train, rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift)


def _prepare_norm(case, g):
    n, d, dt = case["rows"], case["d"], _DTYPES[case["dtype"]]
    s = {"y": _normal(g, n, d).to(dt)}
    if case["residual"] != "none":
        # a residual stream grows over the blocks and has a few channels far above the others
        r = _normal(g, n, d, scale=3.0)
        r[:, :: max(1, d // 3)] *= 20.0
        s["residual"] = r.to(torch.float32 if case["residual"] == "fp32" else dt)
    if case["scale"]:
        s["layer_scale"] = _normal(g, d, scale=0.05, shift=0.1).to(dt)
    if case["gate"]:
        s["gate"] = _normal(g, n, 2 * d).to(dt)[:, d:]   # the gate half of a projection of twice the width
    if case["post"]:
        s["post_w"] = _normal(g, d, scale=0.1, shift=1.0).to(dt)
    if case["next"]:
        s["next_w"] = _normal(g, d, scale=0.1, shift=1.0).to(dt)
    if case["train"]:
        s["d_out"] = _normal(g, n, d).to(s["residual"].dtype if "residual" in s else dt)
        if case["next"]:
            s["d_normed"] = _normal(g, n, d).to(dt)
    return s


def _prepare_route(case, g):
    n, e, dt = case["tokens"], case["experts"], _DTYPES[case["dtype"]]
    popularity = -1.2 * torch.log(torch.randperm(e, generator=g, device="cuda").float() + 1.0)
    scores = _normal(g, n, e, scale=1.5) + (popularity - popularity.mean()) * (1.0 if case["rule"] else 0.1)
    if case["disabled"]:
        off = torch.randperm(e, generator=g, device="cuda")[: case["disabled"]]
        scores[:, off] = -math.inf
    s = {"scores": scores.to(dt), "mask": None}
    if case["padded"]:
        # sequences of one batch, each filled to a length of its own
        length = max(1, -(-n // 8))
        filled = torch.randint(length // 2, length + 1, (8,), generator=g, device="cuda")
        s["mask"] = (torch.arange(length, device="cuda") < filled[:, None]).reshape(-1)[:n].contiguous()
    if case["train"]:
        s["d_gates"] = _normal(g, n, case["k"], scale=1.0 / n)
        s["d_balance"] = torch.full((), BALANCE_WEIGHT, device="cuda")
        s["d_z"] = torch.full((), Z_WEIGHT, device="cuda")
    return s


def _prepare_coef(case, g):
    n, e, k = case["tokens"], case["experts"], case["k"]
    popularity = -1.2 * torch.log(torch.arange(e, device="cuda").float() + 1.0)
    scores = _normal(g, n, e) + (popularity if case["skew"] else 0.0)
    idx = torch.sort(scores, dim=-1, descending=True).indices[:, :k].to(torch.int32)
    gates = torch.rand(n, k, generator=g, device="cuda") + 0.1
    gates /= gates.sum(-1, keepdim=True)
    idx[n - n // 16:] = -1              # padding tokens at the batch's end have no experts
    gates[n - n // 16:] = 0.0
    s = {"idx": idx.contiguous(), "gates": gates.contiguous(), "u": _normal(g, e, case["r1"]).to(_DTYPES[case["dtype"]])}
    if case["train"]:
        s["d_c"] = _normal(g, n, case["r1"])
    return s


def prepare(case, seed):
    make = {"norm": _prepare_norm, "route": _prepare_route, "coef": _prepare_coef}[case["op"]]
    return dict(make(case, _generator(seed)), case=case)


# ---------------------------------------------------------------------------------------------- the framework's own calls
def _own_norm(s):
    from mamba_tuckermoe_b200 import residual_norm
    case = s["case"]
    names = [n for n in ("y", "residual", "layer_scale", "gate", "post_w", "next_w") if n in s]
    t = {n: s[n].detach().requires_grad_() for n in names} if case["train"] else s
    out, normed = residual_norm(t["y"], residual=t.get("residual"), layer_scale=t.get("layer_scale"), gate=t.get("gate"),
                                post_norm=(t["post_w"], EPS) if case["post"] else None,
                                next_norm=(t["next_w"], EPS) if case["next"] else None)
    got = {"out": out, "normed": normed}
    if case["train"]:
        ends, into = [out], [s["d_out"]]
        if normed is not None:
            ends.append(normed)
            into.append(s["d_normed"])
        got.update(zip(("d_" + n for n in names), torch.autograd.grad(ends, [t[n] for n in names], into)))
    return got


def _own_route(s):
    from mamba_tuckermoe_b200 import route_tokens
    case = s["case"]
    scores = s["scores"].detach().requires_grad_() if case["train"] else s["scores"]
    r = route_tokens(scores, case["k"], token_mask=s["mask"], router=(case["rule"], CAP, TEMPERATURE))
    got = {"idx": r.idx, "gates": r.gates, "counts": r.counts, "balance": r.balance_loss, "z": r.z_loss}
    if case["train"]:
        got["d_scores"], = torch.autograd.grad([r.gates, r.balance_loss, r.z_loss], [scores], [s["d_gates"], s["d_balance"], s["d_z"]])
    return got


def _own_coef(s):
    from mamba_tuckermoe_b200 import expert_coefficients
    if not s["case"]["train"]:
        return {"c": expert_coefficients(s["idx"], s["gates"], s["u"])}
    gates, u = s["gates"].detach().requires_grad_(), s["u"].detach().requires_grad_()
    c = expert_coefficients(s["idx"], gates, u)
    d_gates, d_u = torch.autograd.grad(c, [gates, u], s["d_c"])
    return {"c": c, "d_gates": d_gates, "d_u": d_u}


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    case = s["case"]
    y = s["y"].float()
    v, x = y, None
    if case["post"]:
        w0 = s["post_w"].float()
        rho0 = 1.0 / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
        y_hat = y * rho0
        v = y_hat * w0
    if case["gate"]:
        g = s["gate"].float()
        sig = 1.0 / (1.0 + torch.exp(-g))
        x = v
        v = v * (g * sig)
    a = v * s["layer_scale"].float() if case["scale"] else v
    out = s["residual"].float() + a if "residual" in s else a
    out_dtype = s["residual"].dtype if "residual" in s else s["y"].dtype
    got = {"out": out.to(out_dtype), "normed": None}
    if case["next"]:
        w1 = s["next_w"].float()
        rho1 = 1.0 / torch.sqrt((out * out).mean(-1, keepdim=True) + EPS)
        out_hat = out * rho1
        got["normed"] = (out_hat * w1).to(s["y"].dtype)
    if not case["train"]:
        return got
    d_out = s["d_out"].float()
    if case["next"]:
        d_n = s["d_normed"].float()
        got["d_next_w"] = (d_n * out_hat).sum(0).to(s["next_w"].dtype)
        u = w1 * d_n
        d_out = d_out + rho1 * (u - out_hat * (u * out_hat).mean(-1, keepdim=True))
    if "residual" in s:
        got["d_residual"] = d_out.to(out_dtype)
    d_v = d_out
    if case["scale"]:
        got["d_layer_scale"] = (d_out * v).sum(0).to(s["layer_scale"].dtype)
        d_v = d_out * s["layer_scale"].float()
    if case["gate"]:
        got["d_gate"] = (d_v * x * (sig * (1.0 + g * (1.0 - sig)))).to(s["gate"].dtype)
        d_v = d_v * (g * sig)
    if case["post"]:
        got["d_post_w"] = (d_v * y_hat).sum(0).to(s["post_w"].dtype)
        u = w0 * d_v
        d_v = rho0 * (u - y_hat * (u * y_hat).mean(-1, keepdim=True))
    got["d_y"] = d_v.to(s["y"].dtype)
    return got


def _plain_route(s):
    case = s["case"]
    k, e, rule = case["k"], case["experts"], case["rule"]
    raw = s["scores"].float()
    on = raw > -math.inf                                  # an expert whose score is -inf cannot be selected
    token = on.any(-1) if s["mask"] is None else s["mask"] & on.any(-1)
    sel = torch.sort(raw, dim=-1, descending=True, stable=True).indices[:, :k]
    taken = torch.gather(on, 1, sel) & token[:, None]
    idx = torch.where(taken, sel, -1).to(torch.int32)
    if rule:
        th = torch.tanh(raw / CAP)
        logit = torch.where(on, th * (CAP / TEMPERATURE), -math.inf)
    else:
        logit = raw
    top = torch.where(token, logit.amax(-1), 0.0)[:, None]
    ex = torch.where(on & token[:, None], torch.exp(logit - top), 0.0)
    den = torch.where(token[:, None], ex.sum(-1, keepdim=True), 1.0)
    p = ex / den
    lse = torch.where(token, top[:, 0] + torch.log(den[:, 0]), 0.0)
    p_sel = torch.gather(p, 1, sel) * taken
    total = p_sel.sum(-1, keepdim=True)
    gates = p_sel / (total + 1e-6) if rule else p_sel / torch.where(total > 0, total, 1.0)
    if not rule:                                          # softmax over the winners, from their own scores
        won = torch.where(taken, torch.exp(torch.gather(logit, 1, sel) - top), 0.0)
        gates = won / torch.where(token[:, None], won.sum(-1, keepdim=True), 1.0)
    slot = idx.flatten().long() + 1                       # 0: an empty slot
    counts = torch.zeros(e + 1, dtype=torch.int64, device=slot.device).scatter_add_(0, slot, torch.ones_like(slot))[1:]
    n = token.sum().clamp(min=1).float()
    f = counts.float() / (n * k)
    balance = e * (f * (p.double().sum(0) / n)).sum().float()
    z = (lse.double().square().sum() / n).float()
    got = {"idx": idx, "gates": gates, "counts": counts.to(torch.int32), "balance": balance, "z": z}
    if not case["train"]:
        return got
    d_p = (s["d_balance"] * e / n) * f
    d_logit = p * (d_p - (p * d_p).sum(-1, keepdim=True)) + (s["d_z"] * 2.0 / n) * lse[:, None] * p
    inner = (gates * s["d_gates"]).sum(-1, keepdim=True)
    d_logit = d_logit.scatter_add(1, sel, torch.where(taken, gates * (s["d_gates"] - inner), 0.0))
    if rule:
        d_logit = d_logit - p * inner * (1.0 - gates.double().sum(-1, keepdim=True)).float()
        d_logit = d_logit * ((1.0 - th.double().square()) / TEMPERATURE).float()
    got["d_scores"] = torch.where(on & token[:, None], d_logit, 0.0).to(s["scores"].dtype)
    return got


def _plain_coef(s):
    e, u = s["case"]["experts"], s["u"].float()
    live = (s["idx"] >= 0) & (s["idx"] < e)
    row = torch.where(live, s["idx"], 0).long()
    weight = torch.where(live, s["gates"], 0.0)
    picked = u[row]
    got = {"c": (weight[..., None] * picked).sum(1)}
    if s["case"]["train"]:
        got["d_gates"] = torch.where(live, (picked * s["d_c"][:, None, :]).sum(-1), 0.0)
        terms = (weight[..., None] * s["d_c"][:, None, :]).reshape(-1, u.shape[1])
        # long sums over the tokens of popular experts: in 64 bits
        d_u = torch.zeros(u.shape, dtype=torch.float64, device=u.device).index_add_(0, row.reshape(-1), terms.double())
        got["d_u"] = d_u.to(s["u"].dtype)
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "route": _own_route, "coef": _own_coef}[op](state)
    return {"norm": _plain_norm, "route": _plain_route, "coef": _plain_coef}[op](state)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n, d = case["rows"], case["d"]
        rb = 0 if case["residual"] == "none" else 4 if case["residual"] == "fp32" else b
        ob = rb or b
        gate, nxt = (b if case["gate"] else 0), (b if case["next"] else 0)
        params = (int(case["scale"]) + int(case["post"]) + int(case["next"])) * d * b
        # inputs y, residual, gate and the upstream gradients once; out, normed and the gradients once
        per = b + rb + gate + ob + nxt
        flops = 12
        if case["train"]:
            per += ob + nxt + b + rb + gate
            params *= 2
            flops += 24
        return {"bytes": n * d * per + params, "flops": n * d * flops}
    n, e, k = case["tokens"], case["experts"], case["k"]
    if case["op"] == "route":
        bytes_ = n * e * b + n * k * 8 + e * 4 + 8 + (n if case["padded"] else 0)
        flops = n * e * (8 + (8 if case["rule"] else 0))
        if case["train"]:
            bytes_ += n * e * b + n * k * 4 + 8
            flops += n * e * 8
        return {"bytes": bytes_, "flops": flops}
    r1 = case["r1"]
    bytes_, flops = n * k * 8 + e * r1 * b + n * r1 * 4, 2 * n * k * r1
    if case["train"]:
        bytes_ += n * r1 * 4 + n * k * 4 + e * r1 * b
        flops *= 3
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_norm(s):
    case = s["case"]
    t = {n: s[n].double().requires_grad_(case["train"]) for n in ("y", "residual", "layer_scale", "gate", "post_w", "next_w") if n in s}

    def rms(x, w):
        return x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w

    v = rms(t["y"], t["post_w"]) if case["post"] else t["y"]
    if case["gate"]:
        v = v * torch.nn.functional.silu(t["gate"])
    if case["scale"]:
        v = v * t["layer_scale"]
    out = v + t["residual"] if "residual" in t else v
    normed = rms(out, t["next_w"]) if case["next"] else None
    got = {"out": out.detach(), "normed": None if normed is None else normed.detach()}
    if case["train"]:
        loss = (out * s["d_out"].double()).sum()
        if normed is not None:
            loss = loss + (normed * s["d_normed"].double()).sum()
        got.update(zip(("d_" + n for n in t), torch.autograd.grad(loss, list(t.values()))))
    return got


def _exact_route(s):
    case = s["case"]
    k, e, rule = case["k"], case["experts"], case["rule"]
    x = s["scores"].double()
    off = torch.isneginf(x)
    live = ~off.all(-1)
    if s["mask"] is not None:
        live = live & s["mask"]
    order = torch.argsort(-x, dim=-1, stable=True)[:, :k]
    empty = off.gather(1, order) | ~live[:, None]
    rows = live.nonzero()[:, 0]
    # an expert that is off keeps a finite stand-in here and is masked out of every softmax
    leaf = x.masked_fill(off, 0.0)[rows].requires_grad_(case["train"])
    logit = leaf if rule == 0 else CAP * torch.tanh(leaf / CAP) / TEMPERATURE
    logit = logit.masked_fill(off[rows], -math.inf)
    prob = torch.softmax(logit, -1)
    won = logit.gather(1, order[rows]).masked_fill(empty[rows], -math.inf)
    if rule == 0:
        gates = torch.softmax(won, -1)
    else:
        picked = prob.gather(1, order[rows]).masked_fill(empty[rows], 0.0)
        gates = picked / (picked.sum(-1, keepdim=True) + 1e-6)
    counts = torch.zeros(e + 1, dtype=torch.int64, device=x.device)
    counts.scatter_add_(0, torch.where(empty, e, order).reshape(-1), torch.ones_like(order).reshape(-1))
    n = max(1, rows.numel())
    balance = e * torch.dot(counts[:e].double() / (n * k), prob.sum(0) / n)
    z = torch.logsumexp(logit, -1).pow(2).sum() / n
    full = torch.zeros(x.shape[0], k, dtype=torch.float64, device=x.device)
    full[rows] = gates.detach()
    got = {"idx": torch.where(empty, -1, order).to(torch.int32), "gates": full, "counts": counts[:e].to(torch.int32),
           "balance": balance.detach(), "z": z.detach()}
    if case["train"]:
        loss = (gates * s["d_gates"].double()[rows]).sum() + balance * s["d_balance"].double() + z * s["d_z"].double()
        d = torch.zeros_like(x)
        d[rows] = torch.autograd.grad(loss, leaf)[0].masked_fill(off[rows], 0.0)
        got["d_scores"] = d
    return got


def _exact_coef(s):
    case = s["case"]
    n, k, e, r1 = case["tokens"], case["k"], case["experts"], case["r1"]
    gates, u = s["gates"].double(), s["u"].double()
    d_c = s["d_c"].double() if case["train"] else None
    c = torch.zeros(n, r1, dtype=torch.float64, device=u.device)
    d_gates = torch.zeros(n, k, dtype=torch.float64, device=u.device)
    d_u = torch.zeros(e, r1, dtype=torch.float64, device=u.device)
    # expert by expert as dense products with that expert's gate column
    for first in range(0, e, 64):
        ids = torch.arange(first, min(e, first + 64), device=u.device)
        hit = (s["idx"][:, :, None] == ids).double()                    # [n, k, experts of this part]
        dense = (gates[:, :, None] * hit).sum(1)
        c += dense @ u[ids]
        if case["train"]:
            d_gates += (hit * (d_c @ u[ids].t())[:, None, :]).sum(-1)
            d_u[ids] = dense.t() @ d_c
    got = {"c": c}
    if case["train"]:
        got.update(d_gates=d_gates, d_u=d_u)
    return got


def exact(case, seed):
    return {"norm": _exact_norm, "route": _exact_route, "coef": _exact_coef}[case["op"]](prepare(case, seed))
