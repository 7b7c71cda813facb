"""residual_norm, route_tokens and expert_coefficients on the GPU against their float64 statements, element by element within
the bounds that oracle/block_ops_oracle.py derives; gradients also against differences of the float64 forward."""
import pytest
import torch

import mamba_tuckermoe_b200 as pkg
from mamba_tuckermoe_b200 import expert_coefficients, residual_norm, route_tokens
from oracle import block_ops_oracle as ora

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def near(name, got, want):
    value, bound = want
    got = got.detach().double().cpu()
    assert got.shape == value.shape, name
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    over = (got - value).abs() - bound - 1e-37
    assert float(over.max() if over.numel() else 0.0) <= 0.0, \
        f"{name}: off by {float((got - value).abs().max()):.3e}, worst excess {float(over.max()):.3e} of bound {float(bound.flatten()[over.argmax()]):.3e}"


# ------------------------------------------------------------------------------------------------------- residual_norm
def norm_inputs(rows, d, dtype, residual=True, gate=True, scale=True, post=True, nxt=True, res_dtype=None, seed=0, gap=0):
    """CPU tensors; ``gap`` extra columns between rows (0: dense)."""
    g = torch.Generator().manual_seed(seed * 1000 + rows * 7 + d)
    n = lambda *s, a=1.0, b=0.0: torch.randn(*s, generator=g) * a + b
    wide = lambda t: torch.cat([t, torch.full((rows, gap), float("nan"))], 1)[:, :d] if gap else t
    t = {"y": wide(n(rows, d)).to(dtype)}
    t["residual"] = wide(n(rows, d, a=2.0)).to(res_dtype or dtype) if residual else None
    t["gate"] = wide(n(rows, d, a=1.5)).to(dtype) if gate else None
    t["layer_scale"] = n(d, a=0.3, b=0.5).to(dtype) if scale else None
    t["post"] = n(d, a=0.2, b=1.0).to(dtype) if post else None
    t["nxt"] = n(d, a=0.2, b=1.0).to(dtype) if nxt else None
    ups = {"d_out": n(rows, d).to((res_dtype or dtype) if residual else dtype), "d_normed": n(rows, d).to(dtype) if nxt else None}
    return t, ups


def to_gpu(t, gap):
    if t is None:
        return None
    if gap and t.dim() == 2:
        wide = torch.full((t.shape[0], t.shape[1] + gap), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, :t.shape[1]] = t.cuda()
        return wide[:, :t.shape[1]]
    return t.cuda()


def run_norm(t, gap=0, grad=True):
    x = {k: to_gpu(v, gap) for k, v in t.items()}
    if grad:
        x = {k: None if v is None else v.detach().requires_grad_() for k, v in x.items()}
    eps0, eps1 = 1e-5, 2e-5
    out, normed = residual_norm(x["y"], residual=x["residual"], gate=x["gate"], layer_scale=x["layer_scale"],
                                post_norm=None if x["post"] is None else (x["post"], eps0),
                                next_norm=None if x["nxt"] is None else (x["nxt"], eps1))
    return x, out, normed


def check_norm(rows, d, dtype, gap=0, **kw):
    t, ups = norm_inputs(rows, d, dtype, gap=0, **kw)
    want = ora.norm_tail(t["y"], t["residual"], t["gate"], t["layer_scale"], None if t["post"] is None else (t["post"], 1e-5),
                         None if t["nxt"] is None else (t["nxt"], 2e-5), ups["d_out"], ups["d_normed"])
    with torch.no_grad():
        _, out, normed = run_norm(t, gap, grad=False)
    near("out", out, want["out"])
    if normed is not None:
        near("normed", normed, want["normed"])
    x, out_g, normed_g = run_norm(t, gap)
    assert torch.equal(out_g, out) and (normed is None or torch.equal(normed_g, normed))
    names = [k for k, v in x.items() if v is not None]
    ends, into = [out_g], [ups["d_out"].cuda()]
    if normed_g is not None:
        ends.append(normed_g)
        into.append(ups["d_normed"].cuda())
    for k, g in zip(names, torch.autograd.grad(ends, [x[k] for k in names], into)):
        assert g.dtype == x[k].dtype
        near("d_" + k, g, want[k])


@pytest.mark.parametrize("d", [1, 2, 7, 8, 64, 255, 256, 257, 768, 1000, 1001, 1024, 1032, 2048, 2056, 2304, 4608, 5001, 8191, 8192])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_norm_widths(d, dtype):
    check_norm(5, d, dtype)


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 297, 1500])
@pytest.mark.parametrize("d", [40, 768, 1001, 2304])
def test_norm_rows(rows, d):
    check_norm(rows, d, BF)
    if rows <= 297:
        check_norm(rows, d, F32, seed=1)


@pytest.mark.parametrize("flags", range(1, 32))
def test_norm_every_combination_of_operands(flags):
    residual, gate, scale, post, nxt = (bool(flags >> i & 1) for i in range(5))
    kw = dict(residual=residual, gate=gate, scale=scale, post=post, nxt=nxt)
    if not (residual or gate or scale or post):
        kw["scale"] = True
    check_norm(11, 272, BF, **kw)
    check_norm(6, 99, F32, **kw)


@pytest.mark.parametrize("rows,d", [(1, 8), (2, 8), (7, 24), (300, 8), (40000, 128), (2100, 2304), (900, 8192)])
@pytest.mark.parametrize("dtype,res", [(BF, BF), (BF, F32), (F32, F32)])
def test_tail_without_norms(rows, d, dtype, res):
    """One piece a row to 1024, less than a grid of them and several; the last row against rows of a wider tensor too."""
    for kw in (dict(scale=False, gate=False), dict(), dict(scale=False)):
        t, ups = norm_inputs(rows, d, dtype, post=False, nxt=False, res_dtype=res, **kw)
        want = ora.norm_tail(t["y"], t["residual"], t["gate"], t["layer_scale"], None, None, ups["d_out"], None)
        for gap in (0, 8, 3):      # whole pieces, whole pieces apart, and rows that start anywhere (the row walk)
            _, out, normed = run_norm(t, gap=gap, grad=False)
            assert normed is None and out.dtype == res
            near("out", out, want["out"])


def test_tail_without_norms_beyond_32_bit_offsets_and_over_its_residual():
    import ctypes as C
    from mamba_tuckermoe_b200 import _lib
    rows, d = 2 ** 31 // 8192 + 200, 8192
    y = torch.empty(rows, d, dtype=BF, device="cuda")
    y[-200:] = torch.randn(200, d, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    w = torch.rand(d, device="cuda").to(BF)
    out, _ = residual_norm(y, layer_scale=w)
    assert torch.equal(out[-200:], residual_norm(y[-200:].clone(), layer_scale=w)[0])
    del out
    y = y[-200:].clone()
    res = torch.randn(200, d, device="cuda").to(BF)
    want, _ = residual_norm(y, residual=res, layer_scale=w)
    p = _lib.ResidualNorm(200, d, _lib.TMOE_BF16, _lib.TMOE_BF16, 0.0, 0.0, 0, d, d, 0, y.data_ptr(), res.data_ptr(), None, w.data_ptr(), None, None)
    assert _lib.load().tmoe_residual_norm(C.byref(p), res.data_ptr(), None, None, _lib.current_stream_ptr()) == 0 and torch.equal(res, want)


@pytest.mark.parametrize("d", [96, 768, 1003, 2304, 6144])
def test_norm_residual_stream_in_fp32(d):
    check_norm(21, d, BF, res_dtype=F32)
    check_norm(4, d, BF, res_dtype=F32, gate=False, post=False)


@pytest.mark.parametrize("gap", [1, 8, 24])
@pytest.mark.parametrize("d", [256, 770, 1536])
def test_norm_rows_of_a_wider_tensor(gap, d):
    """Row strides other than d, rows that start on odd addresses; the columns in between hold NaN and are not touched."""
    check_norm(13, d, BF, gap=gap)
    check_norm(13, d, F32, gap=gap)


def test_norm_strided_expanded_and_batched_views():
    t, ups = norm_inputs(6, 64, F32)
    # an expanded residual (stride 0), a transposed y (copied), leading batch dimensions, upstream gradients without memory of their own
    res = t["residual"][:1].cuda().expand(6, 64).requires_grad_()
    y = t["y"].cuda().t().contiguous().t().requires_grad_()
    out, normed = residual_norm(y.view(6, 64), residual=res, next_norm=(t["nxt"].cuda(), 1e-5))
    want = ora.norm_tail(t["y"], t["residual"][:1].expand(6, 64), nxt=(t["nxt"], 1e-5), d_out=torch.ones(6, 64), d_normed=torch.ones(6, 64))
    near("out", out, want["out"])
    near("normed", normed, want["normed"])
    (out.sum() + normed.sum()).backward()
    near("d_y", y.grad, want["y"])
    out3, normed3 = residual_norm(t["y"].cuda().view(2, 3, 64), residual=t["residual"].cuda().view(2, 3, 64), next_norm=(t["nxt"].cuda(), 1e-5))
    assert out3.shape == normed3.shape == (2, 3, 64)
    # a leaf that was broadcast over the rows gets the sum over them
    one = t["residual"][0].cuda().requires_grad_()
    out, _ = residual_norm(t["y"].cuda(), residual=one.expand(6, 64))
    out.backward(ups["d_out"].cuda())
    assert torch.allclose(one.grad.cpu(), ups["d_out"].sum(0), atol=1e-5)


def test_norm_only_one_upstream_gradient_and_frozen_inputs():
    t, ups = norm_inputs(7, 320, BF)
    for use in ("d_out", "d_normed"):
        x, out, normed = run_norm(t)
        want = ora.norm_tail(t["y"], t["residual"], t["gate"], t["layer_scale"], (t["post"], 1e-5), (t["nxt"], 2e-5),
                             ups["d_out"] if use == "d_out" else None, ups["d_normed"] if use == "d_normed" else None)
        names = list(x)
        end, up = (out, ups["d_out"]) if use == "d_out" else (normed, ups["d_normed"])
        for k, g in zip(names, torch.autograd.grad(end, [x[k] for k in names], up.cuda(), allow_unused=True)):
            near("d_" + k, g, want[k])
    # only some inputs want gradients
    x = {k: v.cuda() for k, v in t.items()}
    x["layer_scale"].requires_grad_()
    out, normed = residual_norm(x["y"], residual=x["residual"], gate=x["gate"], layer_scale=x["layer_scale"], post_norm=(x["post"], 1e-5),
                                next_norm=(x["nxt"], 2e-5))
    want = ora.norm_tail(t["y"], t["residual"], t["gate"], t["layer_scale"], (t["post"], 1e-5), (t["nxt"], 2e-5), ups["d_out"], None)
    out.backward(ups["d_out"].cuda())
    near("d_layer_scale", x["layer_scale"].grad, want["layer_scale"])
    assert x["y"].grad is None


def test_norm_one_tensor_in_several_places():
    """y as its own residual and gate, one weight in three places: the gradient is the sum of the places'."""
    for dtype in (BF, F32):
        t, ups = norm_inputs(130, 768, dtype)
        x, w = t["y"].cuda(), t["post"].cuda()
        ups = [ups["d_out"].cuda(), ups["d_normed"].cuda()]

        def run(y, residual, gate, scale, post, nxt):
            got = residual_norm(y, residual=residual, gate=gate, layer_scale=scale, post_norm=(post, 1e-6), next_norm=(nxt, 1e-5))
            return got, lambda leaves: torch.autograd.grad(got, leaves, ups)
        y1, w1 = x.clone().requires_grad_(), w.clone().requires_grad_()
        one, grad_one = run(y1, y1, y1, w1, w1, w1)
        many = [a.clone().requires_grad_() for a in (x, x, x, w, w, w)]
        apart, grad_apart = run(*many)
        assert all(torch.equal(a, b) for a, b in zip(one, apart))
        (gy, gw), g = grad_one([y1, w1]), grad_apart(many)
        eps = torch.finfo(dtype).eps          # two additions of autograd's, each rounded by half a step of a partial sum
        for got, parts in ((gy, g[:3]), (gw, g[3:])):
            exact, size = sum(q.double() for q in parts), sum(q.double().abs() for q in parts)
            assert bool(((got.double() - exact).abs() <= size * eps * (1 + eps) + 1e-30).all())


def test_norm_plain_rmsnorm_with_a_gradient():
    """Only next_norm: out is y itself, normed is the layer's own rms_norm to one rounding, and it has a gradient."""
    t, ups = norm_inputs(9, 768, BF, residual=False, gate=False, scale=False, post=False)
    y = t["y"].cuda().requires_grad_()
    out, normed = residual_norm(y, next_norm=(t["nxt"].cuda(), 2e-5))
    assert out is y
    want = ora.norm_tail(t["y"], nxt=(t["nxt"], 2e-5), d_normed=ups["d_normed"])
    near("normed", normed, want["normed"])
    near("rms_norm", pkg.rms_norm(y.detach(), t["nxt"].cuda(), 2e-5), want["normed"])
    normed.backward(ups["d_normed"].cuda())
    near("d_y", y.grad, want["y"])


def test_norm_zero_rows():
    t, ups = norm_inputs(0, 128, BF)
    x, out, normed = run_norm(t)
    assert out.shape == normed.shape == (0, 128)
    (out.sum() + normed.sum()).backward()
    assert x["y"].grad.shape == (0, 128)
    for k in ("layer_scale", "post", "nxt"):
        assert torch.equal(x[k].grad, torch.zeros(128, dtype=BF, device="cuda"))


def test_norm_rows_of_zeros_and_large_values():
    """A row of zeros has rstd = 1/sqrt(eps); rows near the ends of the range stay finite where the formula does."""
    t, ups = norm_inputs(6, 512, F32, gate=False)
    t["y"][1] = 0.0
    t["residual"][1] = 0.0
    t["y"][2] *= 1e15
    t["residual"][3] *= 1e15
    t["y"][4] *= 1e-15
    want = ora.norm_tail(t["y"], t["residual"], None, t["layer_scale"], (t["post"], 1e-5), (t["nxt"], 2e-5), ups["d_out"], ups["d_normed"])
    x, out, normed = run_norm(t)
    near("out", out, want["out"])
    near("normed", normed, want["normed"])
    g = torch.autograd.grad([out, normed], [x["y"], x["residual"]], [ups["d_out"].cuda(), ups["d_normed"].cuda()])
    near("d_y", g[0], want["y"])
    near("d_residual", g[1], want["residual"])


def test_norm_gate_at_its_ends():
    """silu of +-inf-like gates: 0 on the left, g on the right, no NaN from exp overflow."""
    t, ups = norm_inputs(3, 128, F32, post=False)
    t["gate"][0] = -200.0
    t["gate"][1] = 200.0
    want = ora.norm_tail(t["y"], t["residual"], t["gate"], t["layer_scale"], None, (t["nxt"], 2e-5), ups["d_out"], ups["d_normed"])
    x, out, normed = run_norm(t)
    near("out", out, want["out"])
    g, = torch.autograd.grad([out, normed], [x["gate"]], [ups["d_out"].cuda(), ups["d_normed"].cuda()])
    near("d_gate", g, want["gate"])


def test_norm_gradient_against_differences():
    """Directional derivatives of the float64 forward by central differences.  h = 1e-5: truncation ~h^2, cancellation
    ~1e-16 / h = 1e-11; the fp32 kernel's own error is below 1e-5 of the sum's magnitude."""
    t, ups = norm_inputs(4, 96, F32)
    x, out, normed = run_norm(t)
    names = list(x)
    grads = torch.autograd.grad([out, normed], [x[k] for k in names], [ups["d_out"].cuda(), ups["d_normed"].cuda()])

    def loss(v):
        r = ora.norm_tail(v["y"], v["residual"], v["gate"], v["layer_scale"], (v["post"], 1e-5), (v["nxt"], 2e-5))
        return float((r["out"][0] * ups["d_out"]).sum() + (r["normed"][0] * ups["d_normed"]).sum())
    base = {k: v.double() for k, v in t.items()}
    for k, grad in zip(names, grads):
        direction = torch.randn(t[k].shape, generator=torch.Generator().manual_seed(5)).double()
        h = 1e-5
        diff = (loss({**base, k: base[k] + h * direction}) - loss({**base, k: base[k] - h * direction})) / (2 * h)
        terms = grad.double().cpu() * direction
        assert abs(float(terms.sum()) - diff) <= 1e-5 * float(terms.abs().sum()) + 1e-8, k


def test_norm_runs_twice_with_the_same_bits():
    t, ups = norm_inputs(3001, 768, BF)
    got = []
    for _ in range(2):
        x, out, normed = run_norm(t)
        got.append(torch.autograd.grad([out, normed], list(x.values()), [ups["d_out"].cuda(), ups["d_normed"].cuda()]))
    assert all(torch.equal(a, b) for a, b in zip(*got))


# -------------------------------------------------------------------------------------------------------- route_tokens
def route_inputs(T, E, k, dtype, seed=0, spread=1.5, padded=False, off=0):
    g = torch.Generator().manual_seed(seed * 977 + T * 31 + E * 7 + k)
    s = (torch.randn(T, E, generator=g) * spread)
    if off:
        s[torch.rand(T, E, generator=g) < off] = -torch.inf
    mask = torch.rand(T, generator=g) < 0.7 if padded else None
    ups = (torch.randn(T, k, generator=g), torch.tensor(0.7), torch.tensor(0.3))
    return s.to(dtype), mask, ups


def check_route(s, mask, ups, k, rule=0, cap=10.0, temp=0.5):
    want = ora.routing(s, k, mask, (rule, cap, temp), *ups)
    x = s.cuda().requires_grad_()
    m = None if mask is None else mask.cuda()
    r = route_tokens(x, k, token_mask=m, router=(rule, cap, temp))
    assert torch.equal(r.idx.cpu(), want["idx"]) and torch.equal(r.counts.cpu(), want["counts"])
    near("gates", r.gates, want["gates"])
    near("balance", r.balance_loss, want["balance"])
    near("z", r.z_loss, want["z"])
    with torch.no_grad():
        r0 = route_tokens(x, k, token_mask=m, router=(rule, cap, temp))
    assert all(torch.equal(a, b) for a, b in zip(r, r0))
    d, = torch.autograd.grad([r.gates, r.balance_loss, r.z_loss], [x], [u.cuda() for u in ups])
    assert d.dtype == s.dtype
    near("d_scores", d, want["scores"])
    return r


@pytest.mark.parametrize("E", [1, 2, 3, 7, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 128, 250, 256, 257, 512, 520, 1000, 1024])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_route_expert_counts(E, dtype):
    for rule in (0, 1):
        k = min(E, 2 if E % 2 else 8)
        check_route(*route_inputs(19, E, k, dtype), k, rule)


@pytest.mark.parametrize("T", [1, 2, 31, 33, 700, 2500])
@pytest.mark.parametrize("E,k", [(8, 2), (64, 2), (72, 5)])
def test_route_token_counts(T, E, k):
    check_route(*route_inputs(T, E, k, BF, padded=T > 2), k, T % 2)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16])
@pytest.mark.parametrize("E", [16, 24, 60, 96, 200, 300])
def test_route_slots(k, E):
    check_route(*route_inputs(9, E, k, F32), k, 0)
    check_route(*route_inputs(9, E, k, BF, padded=True), k, 1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rule", [0, 1])
def test_route_switched_off_experts_leave_empty_slots(dtype, rule):
    """-inf in most places: rows with fewer experts than slots, rows with none."""
    s, mask, ups = route_inputs(40, 12, 4, dtype, off=0.8, padded=True)
    s[3] = -torch.inf
    mask[3] = True
    s[4] = -torch.inf
    s[4, 7] = 0.25
    mask[4] = True
    r = check_route(s, mask, ups, 4, rule)
    assert r.idx[3].tolist() == [-1] * 4 and r.idx[4].tolist() == [7, -1, -1, -1]
    assert r.gates[3].tolist() == [0.0] * 4


def test_route_no_token_counts():
    for s, mask in ((torch.full((5, 8), -torch.inf), None), (torch.randn(5, 8), torch.zeros(5, dtype=torch.bool)),
                    (torch.randn(0, 8), None)):
        x = s.cuda().requires_grad_()
        r = route_tokens(x, 2, token_mask=None if mask is None else mask.cuda())
        assert bool((r.idx == -1).all()) and float(r.balance_loss) == 0.0 and float(r.z_loss) == 0.0 and int(r.counts.sum()) == 0
        d, = torch.autograd.grad([r.gates, r.balance_loss, r.z_loss], [x], [torch.ones_like(r.gates), torch.ones((), device="cuda"),
                                                                             torch.ones((), device="cuda")])
        assert not bool(d.any())


def test_route_masked_tokens_may_hold_anything():
    """NaN and infinities behind the mask change no bit of the rest and get a zero gradient."""
    for dtype in (BF, F32):
        for rule in (0, 1):
            s, mask, ups = route_inputs(50, 40, 3, dtype, padded=True)
            dirty = s.clone()
            bad = torch.tensor([float("nan"), torch.inf, -torch.inf, torch.finfo(dtype).min])
            dirty[~mask] = bad[torch.arange(40) % 4].to(dtype)
            got = []
            for v in (s, dirty):
                x = v.cuda().requires_grad_()
                r = route_tokens(x, 3, token_mask=mask.cuda(), router=(rule, 10.0, 0.5))
                d, = torch.autograd.grad([r.gates, r.balance_loss, r.z_loss], [x], [u.cuda() for u in ups])
                got.append((*r, d))
            assert all(torch.equal(a, b) for a, b in zip(*got))
            assert not bool(got[1][-1][~mask.cuda()].any())


def test_route_lowest_finite_scores_are_scores():
    """The type's lowest value is a number, not a switch: it is chosen when nothing better is there, and its probability underflows."""
    for dtype in (BF, F32):
        low = torch.finfo(dtype).min
        s = torch.full((3, 10), low).to(dtype)
        s[1, 4] = 0.5
        s[2, 2:5] = torch.tensor([1.0, 2.0, low]).to(dtype)
        r = route_tokens(s.cuda(), 2)
        assert r.idx.tolist() == [[0, 1], [4, 0], [3, 2]]
        assert r.gates[0].tolist() == [0.5, 0.5] and r.gates[1].tolist() == [1.0, 0.0]
        r = route_tokens(s.cuda(), 2, router=(1, 10.0, 0.5))
        assert r.idx.tolist() == [[0, 1], [4, 0], [3, 2]] and bool(torch.isfinite(r.gates).all())


def test_route_caps_far_from_one():
    """Caps so small that finite scores overflow when divided by them (they stay on, at the end of the tanh), and so large that the cap
    does nothing."""
    s, mask, ups = route_inputs(20, 24, 4, F32, spread=1.0)
    s[3, 5], s[3, 6], s[4, 7] = -3e38, 3e38, -3e38
    s[5] = -3e38
    s[6, 2] = -torch.inf
    for cap, temp in ((0.25, 2.0), (1e-3, 0.5)):
        check_route(s, None, ups, 4, 1, cap=cap, temp=temp)
    t, _, ups = route_inputs(20, 24, 4, F32, spread=1.0)
    check_route(t, None, ups, 4, 1, cap=1e6, temp=1.0)


def test_route_ties_signed_zeros_and_nan():
    s = torch.zeros(4, 20)
    s[1, 3:] = -0.0
    s[2, ::2] = 1.0
    s[3, 6] = float("nan")
    s[3, 2] = 5.0
    s[3, 9] = -float("nan")
    for dtype in (BF, F32):
        r = route_tokens(s.to(dtype).cuda(), 3)
        assert r.idx.tolist() == [[0, 1, 2], [0, 1, 2], [0, 2, 4], [6, 9, 2]]
        assert bool(torch.isnan(r.gates[3]).all()) and bool(torch.isnan(r.balance_loss)) and bool(torch.isfinite(r.gates[:3]).all())


def test_route_orders_subnormal_scores():
    for dtype, tiny in ((BF, 2.0 ** -130), (F32, 2.0 ** -140)):
        s = torch.zeros(1, 16)
        s[0, 5], s[0, 9], s[0, 11] = tiny, 2 * tiny, -tiny
        r = route_tokens(s.to(dtype).cuda(), 16)
        assert r.idx[0].tolist() == [9, 5] + [e for e in range(16) if e not in (5, 9, 11)] + [11]


def test_route_saturated_cap():
    """Scores far beyond the cap: the order is still the scores' order, and the gradient's sech^2 keeps its relative accuracy."""
    s, _, ups = route_inputs(12, 48, 4, F32, spread=40.0)
    check_route(s, None, ups, 4, 1)
    check_route(s.to(BF), None, ups, 4, 1, cap=25.0, temp=1.5)


def test_route_rows_of_a_wider_tensor_and_leading_dimensions():
    for E, gap in ((64, 8), (64, 3), (20, 1)):
        for dtype in (BF, F32):
            s, mask, ups = route_inputs(30, E, 2, dtype, padded=True)
            wide = torch.full((30, E + gap), float("nan"), dtype=dtype, device="cuda")
            wide[:, :E] = s.cuda()
            a = route_tokens(wide[:, :E], 2, token_mask=mask.cuda())
            b = route_tokens(s.cuda(), 2, token_mask=mask.cuda())
            assert all(torch.equal(p, q) for p, q in zip(a, b))
            c = route_tokens(s.cuda().view(5, 6, E), 2, token_mask=mask.cuda().view(5, 6))
            assert c.idx.shape == (5, 6, 2) and torch.equal(c.idx.view(30, 2), b.idx) and torch.equal(c.balance_loss, b.balance_loss)


def test_route_each_upstream_gradient_alone():
    s, mask, ups = route_inputs(33, 40, 3, F32, padded=True)
    for rule in (0, 1):
        for i in range(3):
            only = [u if j == i else None for j, u in enumerate(ups)]
            want = ora.routing(s, 3, mask, (rule, 10.0, 0.5), *only)
            x = s.cuda().requires_grad_()
            r = route_tokens(x, 3, token_mask=mask.cuda(), router=(rule, 10.0, 0.5))
            (r.gates, r.balance_loss, r.z_loss)[i].backward(ups[i].cuda())
            near(f"d_scores from output {i}", x.grad, want["scores"])


def test_route_losses_may_be_changed_in_place():
    """The weighted sum of the losses, gathered in place as training code does."""
    s, mask, ups = route_inputs(700, 64, 2, F32, padded=True)
    want = ora.routing(s, 2, mask, (0, 10.0, 0.5), None, torch.tensor(0.5), torch.tensor(0.25))
    x = s.cuda().requires_grad_()
    r = route_tokens(x, 2, token_mask=mask.cuda())
    before = [r.balance_loss.detach().clone(), r.z_loss.detach().clone()]
    loss = r.balance_loss
    loss *= 2.0
    loss += r.z_loss
    r.z_loss.zero_()
    assert torch.equal(loss.detach(), 2.0 * before[0] + before[1])
    loss.backward(torch.tensor(0.25).cuda())
    near("d_scores", x.grad, want["scores"])


def test_route_gradient_against_differences():
    """Central differences of the float64 forward; the scores of one row are more than 2h apart, so no selection changes."""
    s, mask, ups = route_inputs(11, 24, 3, F32, padded=True)
    for rule in (0, 1):
        x = s.cuda().requires_grad_()
        r = route_tokens(x, 3, token_mask=mask.cuda(), router=(rule, 10.0, 0.5))
        grad, = torch.autograd.grad([r.gates, r.balance_loss, r.z_loss], [x], [u.cuda() for u in ups])

        def loss(v):
            w = ora.routing(v, 3, mask, (rule, 10.0, 0.5))
            return float((w["gates"][0] * ups[0]).sum() + ups[1] * w["balance"][0] + ups[2] * w["z"][0])
        direction, h = torch.randn(s.shape, generator=torch.Generator().manual_seed(3)).double(), 1e-6
        assert float((s[:, :, None] - s[:, None, :]).abs().add(torch.eye(24) * 9).min()) > 1e-5
        diff = (loss(s.double() + h * direction) - loss(s.double() - h * direction)) / (2 * h)
        terms = grad.double().cpu() * direction
        assert abs(float(terms.sum()) - diff) <= 2e-5 * float(terms.abs().sum()) + 1e-8


def test_route_agrees_with_the_layers_own_router():
    """From the same scores: the selection of the layer's router kernels, and gates within their rounding to the layer dtype (rule 0
    in bf16: one bf16 rounding of the gate)."""
    from gpu_util import build_module
    from oracle.tucker_moe_oracle import LayerShape, make_factors, make_tokens
    shape = LayerShape(256, 384, 24, 3, 4, 128, 256, 1e-6)
    for dtype in (F32, BF):
        f = make_factors(shape, 5, dtype, 0.05, 0.1)
        # scores that are exact in every accumulation order: small whole numbers
        f["router_w"] = torch.randint(-2, 3, (24, 256), generator=torch.Generator().manual_seed(1)).to(dtype)
        x = torch.zeros(200, 256)
        x[torch.arange(200), torch.arange(200) % 256] = 1.0
        x[torch.arange(200), (torch.arange(200) * 7 + 3) % 256] += 2.0
        x = x.to(dtype).cuda()
        m = build_module(shape, f, dtype)
        _, (idx, gates, c) = m.forward_with_routing(x)
        r = route_tokens(x @ m.router.weight.detach().t(), 3)
        assert torch.equal(r.idx, idx)
        tol = 2 ** -8 if dtype == BF else 1e-5
        assert float(((r.gates - gates).abs() / gates).max()) <= tol


def test_route_runs_twice_with_the_same_bits():
    s, mask, ups = route_inputs(20000, 64, 2, BF, padded=True)
    got = []
    for _ in range(2):
        x = s.cuda().requires_grad_()
        r = route_tokens(x, 2, token_mask=mask.cuda())
        got.append((*r, *torch.autograd.grad([r.gates, r.balance_loss, r.z_loss], [x], [u.cuda() for u in ups])))
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ------------------------------------------------------------------------------------------------- expert_coefficients
def coef_inputs(T, E, k, r1, dtype, seed=0, hot=False, empty=0.1):
    g = torch.Generator().manual_seed(seed + T * 13 + E * 5 + k * 3 + r1)
    idx = torch.randint(0, max(1, E // 16) if hot else E, (T, k), generator=g, dtype=torch.int32)
    bad = torch.tensor([-1, E, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    hole = torch.rand(T, k, generator=g) < empty
    idx[hole] = bad[torch.arange(int(hole.sum())) % 4]
    return idx, torch.rand(T, k, generator=g), torch.randn(E, r1, generator=g).to(dtype), torch.randn(T, r1, generator=g)


def check_coef(idx, gates, u, d_c):
    want = ora.coefficients(idx, gates, u, d_c)
    g, w = gates.cuda().requires_grad_(), u.cuda().requires_grad_()
    c = expert_coefficients(idx.cuda(), g, w)
    near("c", c, want["c"])
    d_g, d_u = torch.autograd.grad(c, [g, w], d_c.cuda())
    near("d_gates", d_g, want["gates"])
    near("d_U", d_u, want["u"])
    assert d_u.dtype == u.dtype


@pytest.mark.parametrize("r1", [1, 2, 3, 4, 7, 8, 16, 31, 32, 33, 64])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_coef_ranks(r1, dtype):
    check_coef(*coef_inputs(45, 12, 3, r1, dtype))


@pytest.mark.parametrize("T", [1, 2, 7, 64, 1000])
@pytest.mark.parametrize("E,k,r1", [(8, 2, 4), (64, 8, 32), (1024, 1, 8), (300, 16, 5)])
def test_coef_sizes(T, E, k, r1):
    check_coef(*coef_inputs(T, E, k, r1, F32, hot=T == 1000))


@pytest.mark.parametrize("k", [1, 2, 3, 4, 8, 9, 16])
@pytest.mark.parametrize("r1", [4, 8, 12, 16, 32, 64])
def test_coef_lane_layouts(k, r1):
    """Every split of a warp into slots and columns, with experts repeated within a token, and enough tokens for several rounds."""
    check_coef(*coef_inputs(203, 9, k, r1, F32))


def test_coef_upstream_gradient_off_16_bytes():
    idx, gates, u, d_c = coef_inputs(77, 40, 2, 8, F32)
    want = ora.coefficients(idx, gates, u, d_c)
    flat = torch.empty(d_c.numel() + 1, device="cuda")
    flat[1:] = d_c.cuda().flatten()
    g, w = gates.cuda().requires_grad_(), u.cuda().requires_grad_()
    d_g, d_u = torch.autograd.grad(expert_coefficients(idx.cuda(), g, w), [g, w], flat[1:].view(77, 8))
    near("d_gates", d_g, want["gates"])
    near("d_U", d_u, want["u"])


def test_coef_many_experts():
    check_coef(*coef_inputs(50, 8192, 2, 4, F32))
    check_coef(*coef_inputs(50, 1024, 2, 64, BF))


def test_coef_same_expert_in_every_slot_and_empty_slots():
    idx, gates, u, d_c = coef_inputs(30, 6, 4, 8, F32, empty=0.0)
    idx[:] = 3
    check_coef(idx, gates, u, d_c)
    idx[:] = -1
    check_coef(idx, gates, u, d_c)
    # an empty slot's gate may hold anything
    gates[:] = float("nan")
    c = expert_coefficients(idx.cuda(), gates.cuda(), u.cuda())
    assert not bool(c.any())


def test_coef_zero_tokens_and_leading_dimensions():
    u = torch.randn(5, 4, device="cuda", requires_grad=True)
    c = expert_coefficients(torch.empty(0, 2, dtype=torch.int32, device="cuda"), torch.empty(0, 2, device="cuda"), u)
    assert c.shape == (0, 4)
    c.sum().backward()
    assert not bool(u.grad.any())
    idx, gates, w, _ = coef_inputs(12, 5, 2, 4, F32)
    a = expert_coefficients(idx.cuda().view(3, 4, 2), gates.cuda().view(3, 4, 2), w.cuda())
    assert a.shape == (3, 4, 4) and torch.equal(a.view(12, 4), expert_coefficients(idx.cuda(), gates.cuda(), w.cuda()))


def test_coef_gradient_against_differences():
    """c is linear in each argument, so a difference of any size is exact up to float64 rounding."""
    idx, gates, u, d_c = coef_inputs(20, 9, 3, 6, F32)
    g, w = gates.cuda().requires_grad_(), u.cuda().requires_grad_()
    d_g, d_u = torch.autograd.grad(expert_coefficients(idx.cuda(), g, w), [g, w], d_c.cuda())
    loss = lambda a, b: float((ora.coefficients(idx, a, b)["c"][0] * d_c).sum())
    for grad, f, at in ((d_g, lambda v: loss(v, u.double()), gates), (d_u, lambda v: loss(gates.double(), v), u)):
        direction = torch.randn(at.shape, generator=torch.Generator().manual_seed(2)).double()
        diff = (f(at.double() + 0.5 * direction) - f(at.double() - 0.5 * direction))
        terms = grad.double().cpu() * direction
        assert abs(float(terms.sum()) - diff) <= 1e-5 * float(terms.abs().sum()) + 1e-10


def test_coef_runs_twice_with_the_same_bits():
    idx, gates, u, d_c = coef_inputs(30000, 16, 2, 8, F32, hot=True)
    got = []
    for _ in range(2):
        g, w = gates.cuda().requires_grad_(), u.cuda().requires_grad_()
        got.append(torch.autograd.grad(expert_coefficients(idx.cuda(), g, w), [g, w], d_c.cuda()))
    assert all(torch.equal(a, b) for a, b in zip(*got))
