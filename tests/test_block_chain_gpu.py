"""The operators around the layer as they are used together: scores -> route_tokens -> expert_coefficients -> the layer's stages ->
residual_norm; the layer's own tails with a norm behind it; and the ways of calling them (streams, threads, captured graphs, the
registered operators)."""
import threading

import pytest
import torch

from gpu_util import build_module
from mamba_tuckermoe_b200 import (PATH_SIMT, expert_coefficients, fused_ffn, fused_out_proj, read_device_status, residual_norm, rms_norm,
                                  route_tokens)
from oracle import block_ops_oracle as ora
from oracle.tucker_moe_oracle import LayerShape, layer_forward_f64, make_factors, make_tokens, rel_fro

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
SHAPE = LayerShape(256, 384, 16, 2, 4, 128, 256, 1e-6)


def make_layer(dtype, shape=SHAPE, seed=5):
    f = make_factors(shape, seed, dtype, 0.1, 0.1)
    return build_module(shape, f, dtype), f


@pytest.mark.parametrize("T", [1, 7, 40, 300])
def test_layer_on_its_own_routing_is_the_layer(T):
    """forward_routed on the coefficients that the layer itself made: the same kernels, so the same bits (CUDA-core path)."""
    m, _ = make_layer(F32)
    x = make_tokens(T, 256, 3, F32).cuda()
    with torch.no_grad():
        y, (idx, gates, c) = m.forward_with_routing(x)
        assert torch.equal(m.forward_routed(x, c), y)
        # and from the indices and gates: at most r1-long fp32 sums apart
        c2 = expert_coefficients(idx, gates, m.U_expert)
        assert torch.allclose(c2, c, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("T", [1, 5, 130, 700])
def test_layer_on_outside_routing_in_bf16(T):
    """Tensor-core stages (also where the layer itself would take its decode kernels) on expert_coefficients of the layer's own choice."""
    m, f = make_layer(BF)
    x = make_tokens(T, 256, 4, BF)
    with torch.no_grad():
        _, (idx, gates, _) = m.forward_with_routing(x.cuda())
        y = m.forward_routed(x.cuda().view(1, T, 256), expert_coefficients(idx, gates, m.U_expert).view(1, T, 4))
    assert y.shape == (1, T, 384)
    y64, _ = layer_forward_f64(x, f, 2, 1e-6, idx=idx.cpu(), round_scores_to=BF)
    assert rel_fro(y[0].float().cpu(), y64) <= 2e-2            # the suite's tolerance of a bf16 layer
    torch.cuda.synchronize()
    assert read_device_status() == (0, 0, 0, 0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_whole_chain(dtype):
    """Scores with one expert switched off and padding masked, through the layer's stages, into a normed, gated residual tail:
    against the float64 chain under the run's own selection."""
    m, f = make_layer(dtype)
    T = 64
    g = torch.Generator().manual_seed(8)
    x = make_tokens(T, 256, 6, dtype)
    mask = torch.arange(T) < 50
    scores = (x.float() @ f["router_w"].float().t()).to(dtype)
    scores[:, 3] = -torch.inf
    rnd = lambda *s: torch.randn(*s, generator=g)
    res, gate, ls = rnd(T, 384).to(dtype), rnd(T, 384).to(dtype), (rnd(384) * 0.1 + 0.5).to(dtype)
    w0, w1 = (rnd(384) * 0.1 + 1).to(dtype), (rnd(384) * 0.1 + 1).to(dtype)
    with torch.no_grad():
        r = route_tokens(scores.cuda(), 2, token_mask=mask.cuda())
        c = expert_coefficients(r.idx, r.gates, m.U_expert)
        y = m.forward_routed(x.cuda(), c)
        out, normed = residual_norm(y, residual=res.cuda(), layer_scale=ls.cuda(), gate=gate.cuda(), post_norm=(w0.cuda(), 1e-5),
                                    next_norm=(w1.cuda(), 1e-5))
    want = ora.routing(scores, 2, mask)
    assert torch.equal(r.idx.cpu(), want["idx"]) and not bool((r.idx == 3).any()) and bool((r.idx[50:] == -1).all())
    assert not bool(c[50:].any())
    c64 = ora.coefficients(want["idx"], want["gates"][0], f["U_expert"])["c"][0]
    h = x.double() @ f["U_in"].double()
    h = h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + 1e-6) * f["inner_norm_w"].double()
    z = torch.einsum("ta,ars,tr->ts", c64, f["core"].double(), h)
    y64 = z @ f["U_out"].double() + f["bias"].double()
    tol = 2e-2 if dtype == BF else 1e-4                        # the suite's tolerances of a layer
    assert rel_fro(y.float().cpu(), y64) <= tol
    # a padded token's layer output is the bias, whatever it holds
    assert rel_fro(y[50:].float().cpu(), f["bias"].double().expand(14, 384)) <= tol
    tail = ora.norm_tail(y.cpu(), res, gate, ls, (w0, 1e-5), (w1, 1e-5))
    for name, got in (("out", out), ("normed", normed)):
        value, bound = tail[name]
        assert bool(((got.double().cpu() - value).abs() <= bound).all()), name


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [2, 90])
def test_layer_tails_with_a_norm_behind_the_layer(dtype, T):
    shape = LayerShape(256, 256, 16, 2, 4, 128, 256, 1e-6)
    m, f = make_layer(dtype, shape)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, 256, generator=g).to(dtype).cuda()
    ls, w0, w1, wp = ((torch.randn(256, generator=g) * 0.1 + 1).to(dtype).cuda() for _ in range(4))
    with torch.no_grad():
        y, routing = m.forward_fused(x, pre_norm=(wp, 1e-5), return_routing=True)
        want = residual_norm(y, residual=x, layer_scale=ls, gate=x, post_norm=(w0, 1e-5), next_norm=(w1, 1e-5))
        kw = dict(pre_norm=(wp, 1e-5), residual=x, layer_scale=ls, silu_gate=x)
        (out, normed), (idx, _, _) = m.forward_fused(x, post_norm=(w0, 1e-5), next_norm=(w1, 1e-5), return_routing=True, **kw)
        assert torch.equal(out, want[0]) and torch.equal(normed, want[1]) and torch.equal(idx, routing[0])
        assert torch.equal(m.forward_fused(x, post_norm=(w0, 1e-5), **kw), m.forward_fused(x, post_norm=(w0, 1e-5), next_norm=(w1, 1e-5), **kw)[0])
        # only the next norm: the epilogue's sum, then the stand-alone norm
        out, normed = m.forward_fused(x, next_norm=(w1, 1e-5), **kw)
        assert torch.equal(out, m.forward_fused(x, **kw)) and torch.equal(normed, rms_norm(out, w1, 1e-5))
        # the block tails pass them on
        a = fused_out_proj(m, x, (wp, 1e-5), ls, post_norm=(w0, 1e-5), next_norm=(w1, 1e-5))
        b = m.forward_fused(x, pre_norm=(wp, 1e-5), residual=x, layer_scale=ls, post_norm=(w0, 1e-5), next_norm=(w1, 1e-5))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        out, normed = fused_ffn(m, m, m, x, (wp, 1e-5), ls, next_norm=(w1, 1e-5))
        assert torch.equal(out, fused_ffn(m, m, m, x, (wp, 1e-5), ls)) and torch.equal(normed, rms_norm(out, w1, 1e-5))
        assert fused_ffn(m, m, m, x, (wp, 1e-5), ls, post_norm=(w0, 1e-5)).shape == x.shape


def test_forward_routed_refuses():
    m, _ = make_layer(F32)
    x = torch.randn(3, 256, device="cuda")
    for c in (torch.zeros(3, 5, device="cuda"), torch.zeros(2, 4, device="cuda"), torch.zeros(3, 4, device="cuda", dtype=BF), torch.zeros(3, 4)):
        with pytest.raises(RuntimeError, match="c must be"):
            m.forward_routed(x, c)
    assert m.forward_routed(x[:0], torch.zeros(0, 4, device="cuda")).shape == (0, 384)


def test_refusals_on_the_gpu():
    y, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    bad = [dict(residual=torch.randn(4, 32, device="cuda")), dict(residual=y.half()), dict(gate=y.bfloat16()), dict(gate=torch.randn(4, 64)),
           dict(layer_scale=w[:32]), dict(layer_scale=w.bfloat16()), dict(next_norm=(w.view(1, 64), 1e-5)), dict(post_norm=(w.cpu(), 1e-5))]
    for kw in bad:
        with pytest.raises(RuntimeError, match="tmoe_b200"):
            residual_norm(y, **kw)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        residual_norm(y.half(), residual=y.half())
    with pytest.raises(RuntimeError, match="does not cover"):
        residual_norm(torch.zeros(1, 8200, device="cuda"), next_norm=(torch.ones(8200, device="cuda"), 1e-5))
    s = torch.randn(5, 8, device="cuda")
    for args, kw in (((s, 9), {}), ((s, 0), {}), ((s.half(), 2), {}), ((s, 2), dict(token_mask=torch.ones(5, device="cuda"))),
                     ((s, 2), dict(token_mask=torch.ones(4, dtype=torch.bool, device="cuda"))), ((s, 2), dict(router=(2, 10.0, 0.5))),
                     ((s, 2), dict(router=(1, 0.0, 0.5))), ((torch.zeros(2, 1025, device="cuda"), 2), {}), ((torch.zeros(2, 64, device="cuda"), 17), {})):
        with pytest.raises(RuntimeError):
            route_tokens(*args, **kw)
    idx, g, u = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, device="cuda"), torch.zeros(4, 4, device="cuda")
    for args in ((idx.long(), g, u), (idx, g.double(), u), (idx, g[:2], u), (idx, g, u.half()), (idx, g, u[0]), (idx.cpu(), g, u),
                 (idx, g, torch.zeros(4, 65, device="cuda"))):
        with pytest.raises(RuntimeError):
            expert_coefficients(*args)


def _chain(y, res, gate, w, scores, u, d_n, d_c):
    """All three operators and their gradients, from fresh leaves."""
    y, res, gate, w, scores, u = (t.detach().requires_grad_() for t in (y, res, gate, w, scores, u))
    out, normed = residual_norm(y, residual=res, gate=gate, post_norm=(w, 1e-5), next_norm=(w, 1e-5))
    r = route_tokens(scores, 3)
    c = expert_coefficients(r.idx, r.gates, u)
    grads = torch.autograd.grad([normed, c, r.balance_loss, r.z_loss], [y, res, gate, w, scores, u],
                                [d_n, d_c, torch.ones_like(r.z_loss), torch.ones_like(r.z_loss)])
    return [t.detach() for t in (out, normed, r.idx, r.gates, r.counts, r.balance_loss, r.z_loss, c)] + list(grads)


def _chain_inputs(seed, rows=777, d=768, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s, t=dtype: torch.randn(*s, generator=g, device="cuda").to(t)
    return (n(rows, d), n(rows, d), n(rows, d), n(d), n(rows, 72), n(72, 8), n(rows, d), n(rows, 8, t=F32))


def test_another_stream_and_two_threads_at_once():
    sets = [_chain_inputs(i) for i in range(4)]
    want = [_chain(*s) for s in sets]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(st):
            for _ in range(10):
                got[i] = _chain(*sets[i])
        st.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_graphs_replayed_side_by_side():
    """Two graphs captured on one stream, replayed at once on two streams with new inputs: they share no scratch."""
    sets = [_chain_inputs(i) for i in range(2)]
    cap = torch.cuda.Stream()
    cap.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(cap):
        for s in sets:
            _chain(*s)
        cap.synchronize()
        for s in sets:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=cap):
                outs.append(_chain(*s))
            graphs.append(g)
    fresh = [_chain_inputs(10 + i) for i in range(2)]
    want = [_chain(*s) for s in fresh]
    for s, f in zip(sets, fresh):
        for a, b in zip(s, f):
            a.copy_(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_calls_do_not_wait_for_the_gpu():
    s = _chain_inputs(1)
    _chain(*s)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        _chain(*s)
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_registered_operators_under_compile():
    """The same results through the registered operators and their gradient formulas (no kernel generator: the aot_eager backend)."""
    y, res, gate, w, scores, u, d_n, d_c = _chain_inputs(3, rows=40)

    def f(y, res, gate, w, scores, u):
        out, normed = residual_norm(y, residual=res, gate=gate, post_norm=(w, 1e-5), next_norm=(w, 1e-5))
        only, _ = residual_norm(y, layer_scale=w)
        r = route_tokens(scores, 3, router=(1, 10.0, 0.5))
        c = expert_coefficients(r.idx, r.gates, u)
        return normed, c, r.balance_loss, r.z_loss, only

    def grads(fn):
        leaves = [t.detach().requires_grad_() for t in (y, res, gate, w, scores, u)]
        o = fn(*leaves)
        g = torch.autograd.grad(o, leaves, [d_n, d_c, torch.ones_like(o[2]), torch.ones_like(o[3]), d_n])
        return [t.detach() for t in o] + list(g)
    a, b = grads(f), grads(torch.compile(f, backend="aot_eager", fullgraph=True))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gradients_of_gradients_are_refused():
    y = torch.randn(4, 64, device="cuda", requires_grad=True)
    s = torch.randn(4, 16, device="cuda", requires_grad=True)
    u = torch.randn(16, 4, device="cuda", requires_grad=True)
    r = route_tokens(s, 2)
    outs = ((residual_norm(y, next_norm=(torch.ones(64, device="cuda"), 1e-5))[1], y), (r.gates.square(), s), (expert_coefficients(r.idx, r.gates, u).square(), u))
    for out, leaf in outs:
        g, = torch.autograd.grad(out.sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="gradients of gradients"):
            (g.sum() + leaf.sum()).backward()


def test_in_place_change_of_a_saved_input_is_noticed():
    y = torch.randn(4, 64, device="cuda", requires_grad=True)
    res = torch.randn(4, 64, device="cuda")
    _, normed = residual_norm(y, residual=res, next_norm=(torch.ones(64, device="cuda"), 1e-5))
    res.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        normed.sum().backward()


def test_rows_beyond_32_bit_offsets():
    """More than 2^31 elements: the last rows come out as a call on them alone gives them."""
    d = 8192
    rows = (1 << 31) // d + 300
    y = torch.empty(rows, d, dtype=BF, device="cuda")
    for i in range(0, rows, 1 << 16):
        y[i:i + (1 << 16)] = torch.arange(i, min(rows, i + (1 << 16)), device="cuda").remainder(97).sub(40).to(BF)[:, None]
    y[:, ::3] *= 0.5
    w = torch.linspace(0.5, 1.5, d, device="cuda").to(BF)
    with torch.no_grad():
        out, normed = residual_norm(y, layer_scale=w, next_norm=(w, 1e-5))
        o, n = residual_norm(y[-500:], layer_scale=w, next_norm=(w, 1e-5))
        assert torch.equal(out[-500:], o) and torch.equal(normed[-500:], n)
        del out, normed
        E = 512
        scores = y.view(-1, E)[: (1 << 31) // E + 1000]
        r = route_tokens(scores, 2)
        q = route_tokens(scores[-1500:], 2)
        assert torch.equal(r.idx[-1500:], q.idx) and torch.equal(r.gates[-1500:], q.gates) and int(r.counts.sum()) == 2 * scores.shape[0]
    del scores, r
    leaf = y.requires_grad_()
    out, _ = residual_norm(leaf, layer_scale=w, post_norm=(w, 1e-5))
    g, = torch.autograd.grad(out, leaf, y.detach())
    tail = y.detach()[-300:].clone().requires_grad_()
    out2, _ = residual_norm(tail, layer_scale=w, post_norm=(w, 1e-5))
    assert torch.equal(g[-300:], torch.autograd.grad(out2, tail, tail.detach())[0])


def test_results_written_over_their_operands():
    """At the C ABI out may be the residual's buffer and normed y's (dense rows)."""
    import ctypes as C
    from mamba_tuckermoe_b200 import _lib
    lib = _lib.load()
    for d, dtype in ((768, BF), (1001, F32), (8192, BF)):
        g = torch.Generator(device="cuda").manual_seed(d)
        y, res = (torch.randn(3000, d, generator=g, device="cuda").to(dtype) for _ in range(2))
        w = torch.rand(d, generator=g, device="cuda").to(dtype)
        want = residual_norm(y, residual=res, post_norm=(w, 1e-5), next_norm=(w, 1e-5))
        dt = _lib.TMOE_BF16 if dtype == BF else _lib.TMOE_F32
        p = _lib.ResidualNorm(3000, d, dt, dt, 1e-5, 1e-5, 0, d, d, 0, y.data_ptr(), res.data_ptr(), None, None, w.data_ptr(), w.data_ptr())
        rc = lib.tmoe_residual_norm(C.byref(p), res.data_ptr(), y.data_ptr(), None, _lib.current_stream_ptr())
        assert rc == 0 and torch.equal(res, want[0]) and torch.equal(y, want[1])


def test_workspace_sizes_are_enough_and_checked():
    """One byte less than the stated workspace is refused; the stated one is never written beyond."""
    import ctypes as C
    from mamba_tuckermoe_b200 import _lib
    lib, st = _lib.load(), _lib.current_stream_ptr()
    for rows, d in ((1, 40), (500, 768), (4000, 2304)):
        y, do = torch.randn(rows, d, device="cuda"), torch.randn(rows, d, device="cuda")
        w, gw, dy = torch.rand(d, device="cuda"), torch.empty(d, device="cuda"), torch.empty(rows, d, device="cuda")
        rstd, n_out = torch.empty(2, rows, device="cuda"), torch.empty(rows, d, device="cuda")
        p = _lib.ResidualNorm(rows, d, 0, 0, 1e-5, 1e-5, 0, d, 0, 0, y.data_ptr(), None, None, None, None, w.data_ptr())
        assert lib.tmoe_residual_norm(C.byref(p), None, n_out.data_ptr(), rstd.data_ptr(), st) == 0
        n = lib.tmoe_residual_norm_workspace_bytes(C.byref(p))
        ws = torch.full((n + 4096,), 171, dtype=torch.uint8, device="cuda")
        args = lambda size: (C.byref(p), rstd.data_ptr(), None, 0, do.data_ptr(), d, dy.data_ptr(), None, None, None, None, gw.data_ptr(), ws.data_ptr(), size, st)
        small = lib.tmoe_residual_norm_backward(*args(n // 2 - 1))
        assert small == -5 and lib.tmoe_residual_norm_backward(*args(n)) == 0
        assert bool((ws[n:] == 171).all())
    for T, E, k in ((5000, 64, 2), (700, 1000, 8), (100000, 8, 1)):
        s = torch.randn(T, E, device="cuda")
        idx, g = torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(T, k, device="cuda")
        cnt, loss = torch.empty(E, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
        p = _lib.Route(T, E, k, 0, 0, 10.0, 0.5, E, s.data_ptr(), None)
        n = lib.tmoe_route_workspace_bytes(C.byref(p))
        ws = torch.full((n + 4096,), 171, dtype=torch.uint8, device="cuda")
        call = lambda size: lib.tmoe_route_tokens(C.byref(p), idx.data_ptr(), g.data_ptr(), cnt.data_ptr(), loss.data_ptr(), None, ws.data_ptr(), size, st)
        assert call(0) == -5 and call(n) == 0 and bool((ws[n:] == 171).all())
    for T, E, k, r1 in ((5000, 64, 2, 4), (900, 1024, 8, 64), (40, 8192, 2, 3)):
        idx = torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda")
        g, u, dc = torch.rand(T, k, device="cuda"), torch.randn(E, r1, device="cuda"), torch.randn(T, r1, device="cuda")
        du = torch.empty_like(u)
        p = _lib.ExpertCoef(T, E, k, r1, 0, idx.data_ptr(), g.data_ptr(), u.data_ptr())
        n = lib.tmoe_expert_coef_workspace_bytes(C.byref(p))
        ws = torch.full((n + 4096,), 171, dtype=torch.uint8, device="cuda")
        call = lambda size: lib.tmoe_expert_coef_backward(C.byref(p), dc.data_ptr(), None, du.data_ptr(), ws.data_ptr(), size, st)
        assert call(0) == -5 and call(n) == 0 and bool((ws[n:] == 171).all())
