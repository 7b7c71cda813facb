"""What residual_norm, route_tokens and expert_coefficients refuse, before anything is enqueued: at the C ABI and in Python; and
the shapes their registered operators promise.  None of this needs a GPU."""
import ctypes as C

import pytest
import torch

import mamba_tuckermoe_b200 as pkg
from mamba_tuckermoe_b200 import _lib
from oracle import block_ops_oracle as ora

P = 4096    # stands for an aligned device pointer: every call here ends before it is used
NULL, SHAPE, DTYPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -5, -6


def norm(**kw):
    base = dict(rows=4, d=64, dtype=1, residual_dtype=1, post_eps=1e-5, next_eps=1e-5, y_stride=64, residual_stride=64, gate_stride=64,
                y=P, residual=P, gate=P, layer_scale=P, post_w=P, next_w=P)
    base.update(kw)
    return _lib.ResidualNorm(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(d=0), SHAPE), (dict(rows=-1), SHAPE), (dict(rows=(1 << 30) + 1), SHAPE), (dict(y_stride=-64), SHAPE),
    (dict(residual_stride=-1), SHAPE), (dict(gate_stride=-1), SHAPE), (dict(d=8193), UNSUPPORTED), (dict(dtype=2), DTYPE),
    (dict(dtype=0, residual_dtype=1), DTYPE), (dict(residual_dtype=7), DTYPE), (dict(residual=None, residual_dtype=0), DTYPE),
    (dict(y=None), NULL), (dict(y=P + 1), ALIGN), (dict(gate=P + 1), ALIGN), (dict(next_w=P + 1), ALIGN),
    (dict(residual_dtype=0, residual=P + 2), ALIGN),
])
def test_norm_refusals(kw, code):
    lib, p = _lib.load(), norm(**kw)
    assert lib.tmoe_residual_norm(C.byref(p), P, P, P, None) == code
    assert lib.tmoe_residual_norm_workspace_bytes(C.byref(p)) == code
    assert lib.tmoe_residual_norm_backward(C.byref(p), P, P, 64, P, 64, P, P, P, P, P, P, P, 1 << 20, None) == code


def test_norm_outputs_and_gradients_that_do_not_belong():
    lib, p = _lib.load(), norm()
    assert lib.tmoe_residual_norm(None, P, P, P, None) == NULL
    assert lib.tmoe_residual_norm(C.byref(p), P, None, P, None) == NULL           # next_w without a place for normed
    assert lib.tmoe_residual_norm(C.byref(norm(next_w=None)), P, P, P, None) == NULL
    assert lib.tmoe_residual_norm(C.byref(norm(next_w=None)), None, None, P, None) == NULL
    assert lib.tmoe_residual_norm(C.byref(p), P + 1, P, P, None) == ALIGN
    assert lib.tmoe_residual_norm(C.byref(norm(rows=0, y=None)), None, None, None, None) == 0
    back = lambda q, rstd=P, do=P, dn=P, dy=P, dr=P, dg=P, dl=P, d0=P, d1=P, ws=P, n=1 << 20, s=64: \
        lib.tmoe_residual_norm_backward(C.byref(q), rstd, do, s, dn, s, dy, dr, dg, dl, d0, d1, ws, n, None)
    assert back(p, do=None, dn=None) == NULL
    assert back(p, rstd=None) == NULL
    assert back(p, s=-1) == SHAPE
    assert back(norm(gate=None)) == NULL and back(norm(residual=None)) == NULL and back(norm(layer_scale=None)) == NULL
    assert back(norm(post_w=None)) == NULL and back(norm(next_w=None)) == NULL
    assert back(norm(next_w=None), d1=None) == NULL                               # d_normed without next_w
    assert back(p, dy=P + 1) == ALIGN and back(p, ws=P + 4) == ALIGN
    assert back(norm(rows=0), dl=None, d0=None, d1=None) == 0
    n = lib.tmoe_residual_norm_workspace_bytes(C.byref(p))
    assert n >= 3 * 64 * 4
    assert lib.tmoe_residual_norm_workspace_bytes(C.byref(norm(rows=0))) == 0


def route(**kw):
    base = dict(tokens=4, n_experts=16, top_k=2, dtype=1, router_mode=0, router_cap=10.0, router_temperature=0.5, scores_stride=16, scores=P,
                token_mask=None)
    base.update(kw)
    return _lib.Route(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), SHAPE), (dict(tokens=(1 << 30) + 1), SHAPE), (dict(n_experts=0), SHAPE), (dict(top_k=0), SHAPE),
    (dict(top_k=17, n_experts=64), SHAPE), (dict(top_k=3, n_experts=2), SHAPE), (dict(scores_stride=-16), SHAPE),
    (dict(n_experts=1025), UNSUPPORTED), (dict(router_mode=2), UNSUPPORTED), (dict(dtype=5), DTYPE), (dict(scores=None), NULL),
    (dict(scores=P + 1), ALIGN), (dict(dtype=0, scores=P + 2), ALIGN), (dict(router_mode=1, router_cap=0.0), SHAPE),
    (dict(router_mode=1, router_cap=float("nan")), SHAPE), (dict(router_mode=1, router_temperature=float("inf")), SHAPE),
    (dict(router_mode=1, router_temperature=-1.0), SHAPE), (dict(router_mode=1, router_cap=1e-39), SHAPE),
    (dict(router_mode=1, router_cap=3e38), SHAPE), (dict(router_mode=1, router_temperature=1e-39), SHAPE),
    (dict(router_mode=1, router_cap=1e25, router_temperature=1e-20), SHAPE), (dict(router_mode=1, router_cap=1e-25, router_temperature=1e20), SHAPE),
])
def test_route_refusals(kw, code):
    lib, p = _lib.load(), route(**kw)
    assert lib.tmoe_route_tokens(C.byref(p), P, P, P, P, P, P, 1 << 20, None) == code
    assert lib.tmoe_route_workspace_bytes(C.byref(p)) == code
    assert lib.tmoe_route_tokens_backward(C.byref(p), P, P, P, P, P, P, P, P, P, None) == code


def test_route_pointers():
    lib, p = _lib.load(), route()
    assert lib.tmoe_route_workspace_bytes(C.byref(p)) == 0                         # one block, no partial sums
    big = route(tokens=100000)
    assert lib.tmoe_route_workspace_bytes(C.byref(big)) > 0
    assert lib.tmoe_route_workspace_bytes(None) == NULL
    for i in (0, 1, 2, 3):                                                        # stats is optional
        args = [P] * 6
        args[i] = None
        assert lib.tmoe_route_tokens(C.byref(p), *args, 1 << 20, None) == NULL
    assert lib.tmoe_route_tokens(C.byref(p), P + 2, P, P, P, P, P, 1 << 20, None) == ALIGN
    assert lib.tmoe_route_tokens(C.byref(p), P, P, P, P, None, P + 4, 1 << 20, None) == ALIGN
    for i in (0, 1, 2, 3, 4, 8):
        args = [P] * 9
        args[i] = None
        assert lib.tmoe_route_tokens_backward(C.byref(p), *args, None) == NULL
    assert lib.tmoe_route_tokens_backward(C.byref(p), P, P, P, P, P, P + 2, P, P, P, None) == ALIGN
    assert lib.tmoe_route_tokens_backward(C.byref(route(tokens=0)), P, P, P, P, P, P, P, P, P, None) == 0


def coef(**kw):
    base = dict(tokens=4, n_experts=16, top_k=2, r1=4, dtype=1, idx=P, gates=P, U_expert=P)
    base.update(kw)
    return _lib.ExpertCoef(**base)


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), SHAPE), (dict(n_experts=0), SHAPE), (dict(top_k=17), SHAPE), (dict(top_k=0), SHAPE), (dict(r1=0), SHAPE),
    (dict(r1=65), SHAPE), (dict(n_experts=8193), UNSUPPORTED), (dict(dtype=9), DTYPE), (dict(idx=None), NULL), (dict(gates=None), NULL),
    (dict(U_expert=None), NULL), (dict(idx=P + 2), ALIGN), (dict(U_expert=P + 1), ALIGN),
])
def test_coef_refusals(kw, code):
    lib, p = _lib.load(), coef(**kw)
    assert lib.tmoe_expert_coef(C.byref(p), P, None) == code
    assert lib.tmoe_expert_coef_workspace_bytes(C.byref(p)) == code
    assert lib.tmoe_expert_coef_backward(C.byref(p), P, P, P, P, 1 << 20, None) == code


def test_coef_pointers():
    lib, p = _lib.load(), coef()
    assert lib.tmoe_expert_coef(C.byref(p), None, None) == NULL
    assert lib.tmoe_expert_coef(C.byref(p), P + 2, None) == ALIGN
    assert lib.tmoe_expert_coef(C.byref(coef(tokens=0)), None, None) == 0
    assert lib.tmoe_expert_coef_backward(C.byref(p), P, None, None, P, 1 << 20, None) == NULL
    assert lib.tmoe_expert_coef_backward(C.byref(p), None, P, P, P, 1 << 20, None) == NULL
    assert lib.tmoe_expert_coef_backward(C.byref(p), P + 2, P, P, P, 1 << 20, None) == ALIGN


def test_python_refuses_cpu_tensors_and_empty_calls():
    y, w = torch.randn(3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.residual_norm(y, next_norm=(w, 1e-5))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.residual_norm(y.requires_grad_(), residual=y)
    with pytest.raises(RuntimeError, match="nothing to do"):
        pkg.residual_norm(y)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.route_tokens(y, 2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        pkg.expert_coefficients(torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2), torch.zeros(4, 4))


def test_fake_operators_give_shapes_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        y, w = torch.empty(2, 5, 64, dtype=torch.bfloat16), torch.empty(64, dtype=torch.bfloat16)
        res = torch.empty(2, 5, 64)
        out, normed, rstd = torch.ops.tmoe_b200.residual_norm(y, res, None, w, None, w, 1e-5, 1e-5)
        assert out.shape == normed.shape == y.shape and out.dtype == torch.float32 and normed.dtype == torch.bfloat16 and rstd.shape == (2, 10)
        g = torch.ops.tmoe_b200.residual_norm_backward(y, res, None, w, None, w, 1e-5, 1e-5, rstd, out, normed)
        assert [t.shape for t in g] == [y.shape, res.shape, w.shape, w.shape]
        idx, gates, counts, losses, stats = torch.ops.tmoe_b200.route_tokens(torch.empty(3, 7, 40), None, 2, 0, 10.0, 0.5)
        assert idx.shape == gates.shape == (3, 7, 2) and idx.dtype == counts.dtype == torch.int32 and counts.shape == (40,) and losses.shape == (3,) and stats.shape == (21, 2)
        assert torch.ops.tmoe_b200.expert_coefficients(idx, gates, torch.empty(40, 6)).shape == (3, 7, 6)


def test_float64_statements_match_autograd():
    """The oracle's hand-written gradients against torch's own of the same float64 formulas."""
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g).double()
    y, r, gt = (rnd(5, 24).requires_grad_() for _ in range(3))
    ls, w0, w1 = (rnd(24).requires_grad_() for _ in range(3))
    rms = lambda x, w, e: x * (x.pow(2).mean(-1, keepdim=True) + e).rsqrt() * w
    out = r + ls * torch.nn.functional.silu(gt) * rms(y, w0, 1e-5)
    normed = rms(out, w1, 1e-5)
    do, dn = rnd(5, 24), rnd(5, 24)
    want = torch.autograd.grad([out, normed], [y, r, gt, ls, w0, w1], [do, dn])
    got = ora.norm_tail(*(t.detach() for t in (y, r, gt, ls)), (w0.detach(), 1e-5), (w1.detach(), 1e-5), do, dn)
    for k, v in zip(("y", "residual", "gate", "layer_scale", "post", "nxt"), want):
        assert torch.allclose(got[k][0], v, rtol=1e-10, atol=1e-12), k
    for rule in (0, 1):
        s, mask, dg = rnd(7, 9), torch.tensor([1, 1, 1, 0, 1, 1, 1]).bool(), rnd(7, 2)
        s[2, 3] = -torch.inf
        o = ora.routing(s, 2, mask, (rule, 10.0, 0.5), dg, torch.tensor(0.5), torch.tensor(0.25))
        x = s.clone().requires_grad_()
        l = 10 * torch.tanh(x / 10) / 0.5 if rule else x
        l = torch.where(torch.isneginf(s), s, l)[mask]
        p, idx = torch.softmax(l, -1), o["idx"][mask].long()
        picked = p.gather(1, idx)
        gates = picked / (picked.sum(-1, keepdim=True) + 1e-6) if rule else torch.softmax(l.gather(1, idx), -1)
        bal = 9 * (o["counts"].double() / 12 * p.mean(0)).sum()
        z = torch.logsumexp(l, -1).pow(2).mean()
        d, = torch.autograd.grad((gates * dg[mask]).sum() + 0.5 * bal + 0.25 * z, x)
        assert torch.allclose(o["gates"][0][mask], gates.detach()) and torch.allclose(o["balance"][0], bal.detach()) and torch.allclose(o["z"][0], z.detach())
        assert torch.allclose(o["scores"][0], torch.where(torch.isneginf(s), torch.zeros(()).double(), d), rtol=1e-9, atol=1e-12)
