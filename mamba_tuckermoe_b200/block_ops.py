"""What stands around a Tucker-MoE layer in its block, forward and backward on B200:

``residual_norm``        the block's tail: norm, gate, layer scale, residual and the next block's norm in one pass
``route_tokens``         top-k routing from scores with a token mask, tokens per expert, balance and z loss
``expert_coefficients``  the coefficient vector ``c[t] = sum_j gates[t, j] * U_expert[idx[t, j]]`` the layer's core takes

All three are differentiable.  They call the C-ABI library on the caller's current stream, allocate their results and scratch
from torch's allocator on it (nothing is kept between calls, so captured graphs share no scratch) and run on CUDA tensors only.
Results are bit-reproducible.  Gradients of gradients are not implemented.  Capture a backward pass on leaves that no eager autograd
graph still holds, as everywhere in torch: the leaves' accumulators belong to the stream of the first graph that uses them.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import ExpertCoef, ResidualNorm, Route

__all__ = ["residual_norm", "route_tokens", "expert_coefficients", "Routing"]

_DTYPES = {torch.float32: _lib.TMOE_F32, torch.bfloat16: _lib.TMOE_BF16}
_is_compiling = torch.compiler.is_compiling
_empty = torch.empty
_F32, _I32, _U8 = torch.float32, torch.int32, torch.uint8


def _fail(what: str):
    raise RuntimeError("tmoe_b200: " + what)


def _call(device: torch.device, name: str, fn, *args):
    """One C entry point on the device's current stream (its last argument).  The raw handle is read without building a Stream object:
    a call at decode sizes costs more here than on the GPU."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc < 0:
        _lib.check(rc, name)


class _FirstOrderOnly(torch.autograd.Function):
    """A gradient that depends on ``anchors`` in a way that has no formula here: differentiating it is an error, not a zero."""

    @staticmethod
    def forward(ctx, grad, *anchors):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        _fail("gradients of gradients are not implemented")


def _first_order(backward):
    """A custom function's backward, whose results refuse to be differentiated where a graph of the gradients is being built."""
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            got = backward(ctx, *grads)
        anchors = [t for t in (*ctx.saved_tensors, *grads) if t is not None and t.requires_grad]
        return tuple(g if g is None else _FirstOrderOnly.apply(g, *anchors) for g in got)
    return run


def _size(name: str, fn, p) -> int:
    n = fn(C.byref(p))
    return n if n >= 0 else _lib.check(n, name)


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """2-D view [rows, width] with contiguous rows (any row stride); copies only what cannot be viewed that way."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if t.stride(1) != 1 and width != 1:
        t = t.contiguous()
    return t


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _like(t: torch.Tensor) -> torch.Tensor:
    """A dense tensor of t's shape and dtype (``empty_like`` of a dense one costs half of ``empty`` with its arguments)."""
    return torch.empty_like(t) if t.is_contiguous() else _empty(t.shape, dtype=t.dtype, device=t.device)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------------- residual_norm
def _check_norm(y, residual, gate, layer_scale, post_w, next_w):
    if not y.is_cuda:
        _fail("residual_norm runs on CUDA tensors only (no CPU fallback)")
    dtype, shape, device = y.dtype, y.shape, y.device
    if dtype not in _DTYPES:
        _fail(f"unsupported dtype {dtype} (float32 and bfloat16 only)")
    if not shape:
        _fail("y must be (..., d)")
    if residual is not None and (residual.shape != shape or residual.device != device or
                                 (residual.dtype != dtype and residual.dtype != _F32)):
        _fail("residual must have y's shape and device and y's dtype or float32")
    if gate is not None and (gate.shape != shape or gate.dtype != dtype or gate.device != device):
        _fail("gate must have y's shape, dtype and device")
    d = shape[-1]
    for w in (layer_scale, post_w, next_w):
        if w is not None and (w.dim() != 1 or w.shape[0] != d or w.dtype != dtype or w.device != device):
            _fail("layer_scale and the norm weights must be (d,) in y's dtype on its device")
    return d


def _norm_struct(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps):
    """(struct, tensors that must outlive the call)"""
    d = y.shape[-1]
    y2 = _rows(y, d)
    dt = _DTYPES[y.dtype]
    res_dt, res_stride, gate_stride, res2, gate2 = dt, 0, 0, None, None
    if residual is not None:
        res2 = _rows(residual, d)
        res_dt, res_stride = _DTYPES[residual.dtype], res2.stride(0)
    if gate is not None:
        gate2 = _rows(gate, d)
        gate_stride = gate2.stride(0)
    keep = [y2, res2, gate2]
    ptrs = []
    for w in (layer_scale, post_w, next_w):
        if w is not None:
            w = _dense(w)
            keep.append(w)
            ptrs.append(w.data_ptr())
        else:
            ptrs.append(None)
    return ResidualNorm(y2.shape[0], d, dt, res_dt, post_eps, next_eps, 0, y2.stride(0), res_stride, gate_stride, y2.data_ptr(),
                        _ptr(res2), _ptr(gate2), *ptrs), keep


def _norm_forward(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps, keep):
    """(out or None, normed or None, rstd or None); out is None where it would be y."""
    _check_norm(y, residual, gate, layer_scale, post_w, next_w)
    p, held = _norm_struct(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps)
    device, out, normed, rstd = y.device, None, None, None
    if residual is not None:
        out = _like(residual)
    elif gate is not None or layer_scale is not None or post_w is not None:
        out = _like(y)
    if next_w is not None:
        normed = _like(y)
    if keep:
        rstd = y.new_empty((2, p.rows), dtype=_F32)
    _call(device, "tmoe_residual_norm", _lib.load().tmoe_residual_norm, C.byref(p), _ptr(out), _ptr(normed), _ptr(rstd))
    return out, normed, rstd


def _norm_backward(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps, rstd, d_out, d_normed, want):
    """Gradients of (y, residual, gate, layer_scale, post_w, next_w) where `want` says so, None elsewhere."""
    p, held = _norm_struct(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps)
    d, device = p.d, y.device
    do2 = dn2 = None
    do_stride = dn_stride = 0
    if d_out is not None:
        do2 = _rows(d_out, d)
        do_stride = do2.stride(0)
    if d_normed is not None:
        dn2 = _rows(d_normed, d)
        dn_stride = dn2.stride(0)
    grads = [_like(t) if w else None for t, w in zip((y, residual, gate, layer_scale, post_w, next_w), want)]
    lib, ws, n = _lib.load(), None, 0
    if want[3] or want[4] or want[5]:
        n = _size("tmoe_residual_norm_workspace_bytes", lib.tmoe_residual_norm_workspace_bytes, p)
        ws = y.new_empty(n, dtype=_U8)
    _call(device, "tmoe_residual_norm_backward", lib.tmoe_residual_norm_backward, C.byref(p), _ptr(rstd), _ptr(do2), do_stride,
          _ptr(dn2), dn_stride, *[None if g is None else g.data_ptr() for g in grads], _ptr(ws), n)
    return grads


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps):
        ctx.set_materialize_grads(False)
        out, normed, rstd = _norm_forward(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps, True)
        ctx.save_for_backward(y, residual, gate, layer_scale, post_w, next_w, rstd)
        ctx.eps = (post_eps, next_eps)
        return out, normed

    @staticmethod
    @_first_order
    def backward(ctx, d_out, d_normed):
        if d_out is None and d_normed is None:
            return (None,) * 8
        *ins, rstd = ctx.saved_tensors
        return (*_norm_backward(*ins, *ctx.eps, rstd, d_out, d_normed, ctx.needs_input_grad[:6]), None, None)


@torch.library.custom_op("tmoe_b200::residual_norm", mutates_args=())
def _residual_norm_op(y: torch.Tensor, residual: Optional[torch.Tensor], gate: Optional[torch.Tensor],
                      layer_scale: Optional[torch.Tensor], post_w: Optional[torch.Tensor], next_w: Optional[torch.Tensor],
                      post_eps: float, next_eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(out, normed, rstd) with an empty tensor for what the call does not make."""
    got = _norm_forward(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps, True)
    return tuple(y.new_empty(0) if t is None else t for t in got)


@_residual_norm_op.register_fake
def _(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps):
    changed = residual is not None or gate is not None or layer_scale is not None or post_w is not None
    out = y.new_empty(y.shape, dtype=y.dtype if residual is None else residual.dtype) if changed else y.new_empty(0)
    normed = y.new_empty(y.shape) if next_w is not None else y.new_empty(0)
    return out, normed, y.new_empty((2, y.numel() // max(y.shape[-1], 1)), dtype=torch.float32)


@torch.library.custom_op("tmoe_b200::residual_norm_backward", mutates_args=())
def _residual_norm_backward_op(y: torch.Tensor, residual: Optional[torch.Tensor], gate: Optional[torch.Tensor],
                               layer_scale: Optional[torch.Tensor], post_w: Optional[torch.Tensor], next_w: Optional[torch.Tensor],
                               post_eps: float, next_eps: float, rstd: torch.Tensor, d_out: Optional[torch.Tensor],
                               d_normed: Optional[torch.Tensor]) -> list[torch.Tensor]:
    ins = (y, residual, gate, layer_scale, post_w, next_w)
    got = _norm_backward(*ins, post_eps, next_eps, rstd, d_out, d_normed, [t is not None for t in ins])
    return [g for g in got if g is not None]


@_residual_norm_backward_op.register_fake
def _(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps, rstd, d_out, d_normed):
    return [t.new_empty(t.shape) for t in (y, residual, gate, layer_scale, post_w, next_w) if t is not None]


def _norm_op_setup(ctx, inputs, output):
    ctx.ins, ctx.eps = inputs[:6], inputs[6:]
    ctx.changed = any(inputs[i] is not None for i in (1, 2, 3, 4))
    ctx.save_for_backward(output[2], *[t for t in ctx.ins if t is not None])
    ctx.has = [t is not None for t in ctx.ins]
    ctx.ins = None


def _norm_op_backward(ctx, d_out, d_normed, d_rstd):
    rstd, *rest = ctx.saved_tensors
    it = iter(rest)
    ins = [next(it) if h else None for h in ctx.has]
    got = iter(_residual_norm_backward_op(*ins, *ctx.eps, rstd, d_out if ctx.changed else None,
                                          d_normed if ctx.has[5] else None))
    return (*[next(got) if h else None for h in ctx.has], None, None)


torch.library.register_autograd("tmoe_b200::residual_norm", _norm_op_backward, setup_context=_norm_op_setup)


def _weight_eps(norm):
    if norm is None:
        return None, 0.0
    if type(norm) is not tuple and hasattr(norm, "weight"):
        return norm.weight, float(norm.eps)
    return norm[0], float(norm[1])


def _wants_grad(*tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def residual_norm(y: torch.Tensor, *, residual: Optional[torch.Tensor] = None, layer_scale: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, post_norm=None, next_norm=None):
    """The tail of a block in one pass: returns ``(out, normed)`` with

        ``out    = residual + layer_scale * silu(gate) * post_norm(y)``
        ``normed = next_norm(out)``

    where every argument but ``y`` is optional and its factor or term is left out without it; ``normed`` is None without
    ``next_norm``, and ``out`` is ``y`` itself where nothing would change it.  Norms are modules with ``.weight`` and ``.eps``
    or ``(weight, eps)`` pairs and mean ``x / sqrt(mean(x^2) + eps) * weight`` (``pure_torch_mlx/model.py:25-27``); the order of
    the factors is the layer's own epilogue's (``model.py:258-260, 340-341``).

    ``y``, ``residual`` and ``gate`` are ``(..., d)`` of one shape, float32 or bfloat16, ``d`` from 1 to 8192; their rows may lie
    any distance apart (a slice of a wider projection, an expanded row).  ``residual`` may be float32 beside bfloat16 blocks, and
    ``out`` has its dtype; ``normed`` and the weights have ``y``'s.  The arithmetic is fp32, ``normed`` comes from the unrounded sum."""
    post_w, post_eps = _weight_eps(post_norm)
    next_w, next_eps = _weight_eps(next_norm)
    changed = residual is not None or gate is not None or layer_scale is not None or post_w is not None
    if not changed and next_w is None:
        _fail("residual_norm has nothing to do: give it a residual, layer_scale, gate, post_norm or next_norm")
    if _is_compiling():
        out, normed, _ = torch.ops.tmoe_b200.residual_norm(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps)
        return out if changed else y, normed if next_w is not None else None
    if torch.is_grad_enabled() and (y.requires_grad or _wants_grad(residual, gate, layer_scale, post_w, next_w)):
        out, normed = _ResidualNorm.apply(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps)
    else:
        out, normed, _ = _norm_forward(y, residual, gate, layer_scale, post_w, next_w, post_eps, next_eps, False)
    return out if changed else y, normed


# -------------------------------------------------------------------------------------------------------- route_tokens
class Routing(NamedTuple):
    """What ``route_tokens`` returns."""
    idx: torch.Tensor           # int32 (..., top_k): experts by descending score; -1 marks an empty slot
    gates: torch.Tensor         # float32 (..., top_k); 0 in an empty slot
    counts: torch.Tensor        # int32 (E,): slots that chose each expert
    balance_loss: torch.Tensor  # float32 scalar: E * sum_e f_e P_e
    z_loss: torch.Tensor        # float32 scalar: mean of logsumexp(logits)^2


def _check_route(scores, top_k, mask):
    if not scores.is_cuda:
        _fail("route_tokens runs on CUDA tensors only (no CPU fallback)")
    if scores.dtype not in _DTYPES:
        _fail(f"unsupported dtype {scores.dtype} (float32 and bfloat16 only)")
    if scores.dim() == 0 or not 0 < top_k <= scores.shape[-1]:
        _fail(f"scores must be (..., E) with top_k={top_k} in 1..E")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != scores.shape[:-1] or mask.device != scores.device):
        _fail("token_mask must be a bool tensor of scores.shape[:-1] on its device")


def _route_struct(scores, mask, top_k, router):
    """(struct, tensors that must outlive the call)"""
    E = scores.shape[-1]
    s2 = _rows(scores, E)
    if mask is not None:
        mask = _dense(mask)
    return Route(s2.shape[0], E, top_k, _DTYPES[s2.dtype], router[0], router[1], router[2], s2.stride(0), s2.data_ptr(),
                 _ptr(mask)), (s2, mask)


def _route_forward(scores, mask, top_k, router, keep=False):
    """(idx, gates, counts, losses, stats or None)"""
    _check_route(scores, top_k, mask)
    p, held = _route_struct(scores, mask, top_k, router)
    slots, dev = (*scores.shape[:-1], top_k), scores.device
    idx = scores.new_empty(slots, dtype=_I32)
    gates = torch.empty_like(idx, dtype=_F32)
    counts = scores.new_empty(scores.shape[-1], dtype=_I32)
    losses = scores.new_empty(3, dtype=_F32)
    stats = scores.new_empty((p.tokens, 2), dtype=_F32) if keep else None
    lib = _lib.load()
    n = _size("tmoe_route_workspace_bytes", lib.tmoe_route_workspace_bytes, p)
    ws = scores.new_empty(n, dtype=_U8) if n else None
    _call(dev, "tmoe_route_tokens", lib.tmoe_route_tokens, C.byref(p), idx.data_ptr(), gates.data_ptr(), counts.data_ptr(),
          losses.data_ptr(), _ptr(stats), _ptr(ws), n)
    return idx, gates, counts, losses, stats


def _route_backward(scores, mask, idx, gates, counts, losses, stats, top_k, router, d_gates, d_balance, d_z):
    p, held = _route_struct(scores, mask, top_k, router)
    if d_gates is not None:
        d_gates = _dense(d_gates)
    d_scores = _like(scores)
    _call(scores.device, "tmoe_route_tokens_backward", _lib.load().tmoe_route_tokens_backward, C.byref(p), idx.data_ptr(),
          gates.data_ptr(), counts.data_ptr(), losses.data_ptr(), stats.data_ptr(), _ptr(d_gates), _ptr(d_balance), _ptr(d_z),
          d_scores.data_ptr())
    return d_scores


class _RouteTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, mask, top_k, router):
        ctx.set_materialize_grads(False)
        idx, gates, counts, losses, stats = _route_forward(scores, mask, top_k, router, True)
        ctx.mark_non_differentiable(idx, counts)
        ctx.save_for_backward(scores, mask, idx, gates, counts, losses, stats)
        ctx.top_k, ctx.router = top_k, router
        # .data: results of their own, not views of a saved tensor, so that `loss += ...` may change them in place (the backward call reads
        # the token count behind them only)
        return idx, gates, counts, losses[0].data, losses[1].data

    @staticmethod
    @_first_order
    def backward(ctx, d_idx, d_gates, d_counts, d_balance, d_z):
        if d_gates is None and d_balance is None and d_z is None:
            return None, None, None, None
        return _route_backward(*ctx.saved_tensors, ctx.top_k, ctx.router, d_gates, d_balance, d_z), None, None, None


@torch.library.custom_op("tmoe_b200::route_tokens", mutates_args=())
def _route_tokens_op(scores: torch.Tensor, mask: Optional[torch.Tensor], top_k: int, router_mode: int, router_cap: float,
                     router_temperature: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(idx, gates, counts, losses, stats); losses = balance, z and the number of tokens that count."""
    return _route_forward(scores, mask, top_k, (router_mode, router_cap, router_temperature), True)


@_route_tokens_op.register_fake
def _(scores, mask, top_k, router_mode, router_cap, router_temperature):
    return (scores.new_empty((*scores.shape[:-1], top_k), dtype=torch.int32),
            scores.new_empty((*scores.shape[:-1], top_k), dtype=torch.float32),
            scores.new_empty((scores.shape[-1],), dtype=torch.int32), scores.new_empty((3,), dtype=torch.float32),
            scores.new_empty((scores.numel() // max(scores.shape[-1], 1), 2), dtype=torch.float32))


@torch.library.custom_op("tmoe_b200::route_tokens_backward", mutates_args=())
def _route_tokens_backward_op(scores: torch.Tensor, mask: Optional[torch.Tensor], idx: torch.Tensor, gates: torch.Tensor,
                              counts: torch.Tensor, losses: torch.Tensor, stats: torch.Tensor, top_k: int, router_mode: int, router_cap: float,
                              router_temperature: float, d_gates: torch.Tensor, d_losses: torch.Tensor) -> torch.Tensor:
    return _route_backward(scores, mask, idx, gates, counts, losses, stats, top_k, (router_mode, router_cap, router_temperature), d_gates,
                           d_losses[0], d_losses[1])


@_route_tokens_backward_op.register_fake
def _(scores, mask, idx, gates, counts, losses, stats, top_k, router_mode, router_cap, router_temperature, d_gates, d_losses):
    return scores.new_empty(scores.shape)


def _route_op_setup(ctx, inputs, output):
    scores, mask, *rule = inputs
    ctx.rule, ctx.has_mask = rule, mask is not None
    ctx.save_for_backward(scores, *output, *([mask] if mask is not None else []))
    ctx.mark_non_differentiable(output[0], output[2], output[4])


def _route_op_backward(ctx, d_idx, d_gates, d_counts, d_losses, d_stats):
    scores, idx, gates, counts, losses, stats, *mask = ctx.saved_tensors
    d = torch.ops.tmoe_b200.route_tokens_backward(scores, mask[0] if mask else None, idx, gates, counts, losses, stats, *ctx.rule, d_gates, d_losses)
    return (d, None, None, None, None, None)


torch.library.register_autograd("tmoe_b200::route_tokens", _route_op_backward, setup_context=_route_op_setup)


def route_tokens(scores: torch.Tensor, top_k: int, *, token_mask: Optional[torch.Tensor] = None,
                 router=(0, 10.0, 0.5)) -> Routing:
    """Routing of tokens from their router scores ``(..., E)``, differentiable in the scores; returns a ``Routing``.

    ``router`` is the layer's ``(mode, cap, temperature)``: rule 0 takes the softmax over the winners' raw scores
    (``pure_torch_mlx/model.py:75-77``), rule 1 the capped, tempered softmax over all experts, renormalised over the winners
    (``sft_cot_bundle/scripts/model.py:318-329``).  With ``p`` = softmax of the logits over all experts, ``n`` the tokens that count
    and ``f_e = counts_e / (n top_k)``: ``balance_loss = E * sum_e f_e * mean_t p[t, e]`` (1 for uniform routing; the counts carry no
    gradient) and ``z_loss = mean_t logsumexp(logits[t])^2``.

    ``token_mask`` (bool, ``scores.shape[:-1]``): tokens that are False (padding) get empty slots and count nowhere; their
    scores are not used and get no gradient.  A score of ``-inf`` switches an expert off for a token.  Equal scores go to the lower
    expert.  E up to 1024, ``top_k`` up to 16.  fp32 arithmetic whatever the scores' dtype; the layer's bf16 kernels round rule-1
    logits to bf16, this function does not."""
    top_k, router = int(top_k), (int(router[0]), float(router[1]), float(router[2]))
    if _is_compiling():
        idx, gates, counts, losses, _ = torch.ops.tmoe_b200.route_tokens(scores, token_mask, top_k, *router)
        return Routing(idx, gates, counts, losses[0], losses[1])
    if scores.requires_grad and torch.is_grad_enabled():
        return Routing(*_RouteTokens.apply(scores, token_mask, top_k, router))
    idx, gates, counts, losses, _ = _route_forward(scores, token_mask, top_k, router)
    return Routing(idx, gates, counts, losses[0], losses[1])


# ------------------------------------------------------------------------------------------------- expert_coefficients
def _check_coef(idx, gates, U_expert):
    if not U_expert.is_cuda:
        _fail("expert_coefficients runs on CUDA tensors only (no CPU fallback)")
    if U_expert.dtype not in _DTYPES or U_expert.dim() != 2:
        _fail("U_expert must be (E, r1) in float32 or bfloat16")
    if idx.dtype != torch.int32 or gates.dtype != torch.float32 or idx.dim() == 0 or idx.shape != gates.shape:
        _fail("idx (int32) and gates (float32) must be (..., top_k) of one shape")
    if idx.device != U_expert.device or gates.device != U_expert.device:
        _fail("idx, gates and U_expert must be on one device")


def _coef_struct(idx, gates, u):
    """(struct, tensors that must outlive the call)"""
    idx, gates, u = _dense(idx), _dense(gates), _dense(u)
    k = idx.shape[-1]
    return ExpertCoef(idx.numel() // k if k else 0, u.shape[0], k, u.shape[1], _DTYPES[u.dtype], idx.data_ptr(), gates.data_ptr(),
                      u.data_ptr()), (idx, gates, u)


def _coef_forward(idx, gates, u):
    _check_coef(idx, gates, u)
    p, held = _coef_struct(idx, gates, u)
    c = gates.new_empty((*idx.shape[:-1], u.shape[1]))
    _call(u.device, "tmoe_expert_coef", _lib.load().tmoe_expert_coef, C.byref(p), c.data_ptr())
    return c


def _coef_backward(idx, gates, u, d_c, want_gates, want_u):
    p, held = _coef_struct(idx, gates, u)
    d_c, dev = _dense(d_c), u.device
    d_gates = _like(gates) if want_gates else None
    lib, d_u, ws, n = _lib.load(), None, None, 0
    if want_u:
        d_u = _like(u)
        n = _size("tmoe_expert_coef_workspace_bytes", lib.tmoe_expert_coef_workspace_bytes, p)
        ws = u.new_empty(n, dtype=_U8)
    _call(dev, "tmoe_expert_coef_backward", lib.tmoe_expert_coef_backward, C.byref(p), d_c.data_ptr(), _ptr(d_gates), _ptr(d_u),
          _ptr(ws), n)
    return d_gates, d_u


class _ExpertCoefficients(torch.autograd.Function):
    @staticmethod
    def forward(ctx, idx, gates, u):
        ctx.save_for_backward(idx, gates, u)
        return _coef_forward(idx, gates, u)

    @staticmethod
    @_first_order
    def backward(ctx, d_c):
        return (None, *_coef_backward(*ctx.saved_tensors, d_c, ctx.needs_input_grad[1], ctx.needs_input_grad[2]))


@torch.library.custom_op("tmoe_b200::expert_coefficients", mutates_args=())
def _coef_op(idx: torch.Tensor, gates: torch.Tensor, U_expert: torch.Tensor) -> torch.Tensor:
    return _coef_forward(idx, gates, U_expert)


@_coef_op.register_fake
def _(idx, gates, U_expert):
    return gates.new_empty((*idx.shape[:-1], U_expert.shape[1]), dtype=torch.float32)


@torch.library.custom_op("tmoe_b200::expert_coefficients_backward", mutates_args=())
def _coef_backward_op(idx: torch.Tensor, gates: torch.Tensor, U_expert: torch.Tensor, d_c: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    return _coef_backward(idx, gates, U_expert, d_c, True, True)


@_coef_backward_op.register_fake
def _(idx, gates, U_expert, d_c):
    return gates.new_empty(gates.shape), U_expert.new_empty(U_expert.shape)


def _coef_op_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _coef_op_backward(ctx, d_c):
    return (None, *torch.ops.tmoe_b200.expert_coefficients_backward(*ctx.saved_tensors, d_c))


torch.library.register_autograd("tmoe_b200::expert_coefficients", _coef_op_backward, setup_context=_coef_op_setup)


def expert_coefficients(idx: torch.Tensor, gates: torch.Tensor, U_expert: torch.Tensor) -> torch.Tensor:
    """``c[t] = sum_j gates[t, j] * U_expert[idx[t, j]]`` in float32, ``(..., r1)``: the coefficients that mix the layer's core slices
    (``pure_torch_mlx/model.py:93``), for ``TuckerMoE.forward_routed``; differentiable in ``gates`` and ``U_expert``.

    ``idx`` int32 and ``gates`` float32 ``(..., top_k)`` as ``route_tokens`` or ``forward_with_routing`` return them; a slot whose index
    lies outside ``0 .. E-1`` (an empty slot's is -1) adds nothing.  The same expert may appear in several slots of a token.
    ``U_expert`` ``(E, r1)``, E up to 8192, r1 up to 64, ``top_k`` up to 16."""
    if _is_compiling():
        return torch.ops.tmoe_b200.expert_coefficients(idx, gates, U_expert)
    if torch.is_grad_enabled() and (gates.requires_grad or U_expert.requires_grad):
        return _ExpertCoefficients.apply(idx, gates, U_expert)
    return _coef_forward(idx, gates, U_expert)
