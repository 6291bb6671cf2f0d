"""linear_act against the formula in 64 bits.

Tolerances.  A sum of K products in fp32 errs by at most K/2^23 of the sum of
the magnitudes when every add may round by a whole unit; tiles and tensor
instructions add in far fewer steps, so a quarter of that (plus 16 steps for
short sums) is allowed.  A 16-bit output adds half its unit (2^-9 or 2^-12
relative; twice that is allowed), a 16-bit gradient enters its product through
two roundings more.  Activations and their derivatives move by at most twice
their argument's error."""

import math

import pytest
import torch

from stockfish_trainer_b200.layer_stacks import ACTIVATIONS, _native, linear_act

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12}
TYPES = list(UNIT)


def _act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "crelu":
        return z.clamp(0, 1)
    if name == "sqr_crelu":
        return z.clamp(0, 1) ** 2
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z * math.sqrt(0.5))  # exact in the lower tail too
    return z


def _acc(k):
    return (k / 4 + 16) * 2.0**-23


def _grid(shape, g, dt):
    """Multiples of 1/4 in [-1, 1]: products are multiples of 1/16, exact in
    every type and order."""
    return (torch.randint(-4, 5, shape, generator=g) / 4).to(dt)


def _check(got, want, tol):
    assert got.shape == want.shape
    err = (got.double().cpu() - want).abs()
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp_min(1e-300)).max()):.3g} x tol"


def _run(x, w, b, r, act, go, grid=False):
    """Compares the output and every gradient; returns nothing."""
    dt, u, K, N, M = x.dtype, UNIT[x.dtype], x.shape[1], w.shape[0], x.shape[0]
    ref = [t.detach().double().cpu().requires_grad_() if t is not None else None for t in (x, w, b, r)]
    z = ref[0] @ ref[1].t() + (ref[2] if b is not None else 0)
    o = _act(z, act) + (ref[3] if r is not None else 0)
    leaves = [t.detach().clone().requires_grad_() if t is not None else None for t in (x, w, b, r)]
    for have, t in zip(leaves, (x, w, b, r)):
        if have is not None and t.stride() != have.stride():
            have.data = t.detach()
    out = linear_act(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act)
    assert out.dtype == dt
    mag = x.double().cpu().abs() @ w.double().cpu().abs().t() + (b.double().cpu().abs() if b is not None else 0)
    zerr = torch.zeros_like(mag) if grid else mag * _acc(K)
    _check(out, o.detach(), 2 * u * o.detach().abs() + 2 * zerr + 1e-30 + 4 * u * mag * (dt == torch.float32) +
           (r.double().cpu().abs() * 2 * u if r is not None else 0) + (6e-8 if dt == torch.float16 else 0))
    used = [t for t in leaves if t is not None]
    got = torch.autograd.grad(out, used, go)
    dz = torch.autograd.grad(o, z, go.double().cpu(), retain_graph=True)[0]
    want = torch.autograd.grad(o, [t for t in ref if t is not None], go.double().cpu())
    # dz itself: two roundings and the derivative's error from z; the derivative is bounded by 2.2
    gabs = go.double().cpu().abs()
    dzerr = 3 * u * gabs * 2.2 + 2 * zerr * gabs + (1e-7 * gabs if dt == torch.float16 else 0)
    dzabs = dz.abs() + dzerr
    wabs, xabs = w.double().cpu().abs(), x.double().cpu().abs()
    tiny = 6e-8 if dt == torch.float16 else 1e-30
    tols = [dzerr @ wabs + _acc(N) * (dzabs @ wabs) + 2 * u * want[0].abs() + tiny,
            dzerr.t() @ xabs + _acc(M) * (dzabs.t() @ xabs) + 2 * u * want[1].abs() + tiny]
    if b is not None:
        bu = UNIT[b.dtype]
        tols.append(dzerr.sum(0) + _acc(M) * dzabs.sum(0) + 2 * bu * want[2].abs() + tiny)
    if r is not None:
        tols.append(torch.zeros_like(gabs))
    for g, wnt, t in zip(got, want, tols):
        _check(g, wnt, t)


def _make(M, K, N, dt, seed, bias=True, residual=True, bias_f32=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).to(dt)
    w = (torch.randn(N, K, generator=g) / math.sqrt(K)).to(dt)
    b = (0.3 * torch.randn(N, generator=g)).to(torch.float32 if bias_f32 else dt) if bias else None
    r = torch.randn(M, N, generator=g).to(dt) if residual else None
    go = torch.randn(M, N, generator=g).to(dt)
    return [t.cuda() if t is not None else None for t in (x, w, b, r, go)]


SIZES = [(1, 1, 1), (1, 1040, 256), (3, 17, 5), (7, 64, 1), (8, 1040, 32), (24, 1040, 1040), (33, 65, 129),
         (128, 64, 256), (129, 63, 257), (130, 520, 208), (257, 1040, 16), (500, 8, 260), (1000, 331, 517)]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_sizes(cuda, M, K, N, dt):
    x, w, b, r, go = _make(M, K, N, dt, seed=M + K + N)
    _run(x, w, b, r, "silu", go)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_long_sums(cuda, dt):
    """Many rows: the weight gradient's sum is the long one; ragged everywhere."""
    x, w, b, r, go = _make(20011, 72, 24, dt, seed=5, residual=False)
    _run(x, w, b, r, "gelu", go)
    x, w, b, r, go = _make(40, 9000, 136, dt, seed=6, residual=False)
    _run(x, w, b, r, "none", go)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("act", ACTIVATIONS)
def test_activations_on_a_grid(cuda, act, dt):
    """z is a multiple of 1/16 plus 1/32: exact, and never on a kink."""
    g = torch.Generator().manual_seed(3)
    x, w = _grid((150, 40), g, dt), _grid((70, 40), g, dt)
    b = (torch.randint(-8, 9, (70,), generator=g) / 16 + 1 / 32).to(dt)
    go = torch.randn(150, 70, generator=g).to(dt)
    _run(x.cuda(), w.cuda(), b.cuda(), None, act, go.cuda(), grid=True)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_grid_products_are_exact(cuda, dt):
    """No rounding happens anywhere: any misplaced element shows as a whole step."""
    g = torch.Generator().manual_seed(4)
    x, w = _grid((261, 200), g, dt).cuda(), _grid((150, 200), g, dt).cuda()
    out = linear_act(x.float(), w.float()) if dt == torch.float32 else linear_act(x, w)
    want = (x.double() @ w.double().t())
    assert torch.equal(out, want.to(dt))


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_derivatives_at_the_kinks_are_zero(cuda, dt):
    x = torch.tensor([[0.0], [1.0], [-0.0], [0.5], [2.0], [-1.0]], device=cuda, dtype=dt)
    w = torch.ones(1, 1, device=cuda, dtype=dt)
    for act, want in (("relu", [0, 1, 0, 1, 1, 0]), ("crelu", [0, 0, 0, 1, 0, 0]), ("sqr_crelu", [0, 0, 0, 1, 0, 0])):
        xx = x.clone().requires_grad_()
        linear_act(xx, w, activation=act).sum().backward()
        assert xx.grad.flatten().tolist() == want, act


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_extreme_arguments(cuda, dt):
    """The smooth activations at arguments where a factor under- or overflows."""
    z = torch.tensor([-90.0, -20.0, -6.0, -1e-4, 0.0, 1e-4, 6.0, 20.0, 90.0, 3e4], device=cuda).to(dt)
    for act in ("silu", "gelu"):
        x = z[:, None].clone().requires_grad_()
        out = linear_act(x, torch.ones(1, 1, device=cuda, dtype=dt), activation=act)
        out.sum().backward()
        ref = z.double().requires_grad_()
        want = _act(ref, act)
        want.sum().backward()
        # near 0 a product's relative error counts, in the tails the absolute one
        u = 4 * UNIT[dt] + 4e-7
        for got, exp in ((out.flatten(), want.detach()), (x.grad.flatten(), ref.grad)):
            assert ((got.double() - exp).abs() <= u * exp.abs() + 1e-6).all(), (act, got, exp)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_layouts(cuda, dt):
    """Row strides, offsets that break alignment, transposed operands, extra dimensions, broadcast residual and
    gradient, a bias in 32 bits: all equal the plain layout's result bit for bit."""
    x, w, b, r, go = _make(70, 48, 40, dt, seed=9)
    want = linear_act(x, w, b, residual=r, activation="silu")
    for pad, off in ((8, 0), (1, 0), (3, 1), (0, 1), (16, 8)):
        def view(t):
            buf = torch.full((t.shape[0] * (t.shape[1] + pad) + off,), float("nan"), device=cuda, dtype=dt)
            v = buf[off:].view(t.shape[0], -1)[:, :t.shape[1]]
            v.copy_(t)
            return v

        got = linear_act(view(x), view(w), b, residual=view(r), activation="silu")
        torch.testing.assert_close(got, want, rtol=2 * UNIT[dt], atol=1e-6)
        _run(view(x), view(w), b, view(r), "silu", view(go))
    xt, wt = x.t().contiguous().t(), w.t().contiguous().t()
    assert torch.equal(linear_act(xt, wt, b, residual=r, activation="silu"), want)
    got = linear_act(x.view(7, 10, 48), w, b, residual=r.view(7, 10, 40), activation="silu")
    assert got.shape == (7, 10, 40) and torch.equal(got.view(70, 40), want)
    assert linear_act(x[0], w, b).shape == (40,)
    rr = torch.randn(40, device=cuda).to(dt).requires_grad_()
    ww = w.clone().requires_grad_()
    out = linear_act(x, ww, b, residual=rr)
    out.sum().backward()  # a gradient of stride 0
    assert rr.grad.shape == (40,) and (rr.grad == 70).all()
    err = (ww.grad.double() - x.double().sum(0)).abs()
    assert (err <= _acc(70) * x.double().abs().sum(0) + 2 * UNIT[dt] * x.double().sum(0).abs()).all()
    if dt != torch.float32:
        x, w, b, r, go = _make(33, 48, 40, dt, seed=10, bias_f32=True)
        _run(x, w, b, r, "silu", go)


def test_selected_gradients(cuda):
    """Only what is asked for is computed, and it does not depend on the rest."""
    x, w, b, r, go = _make(65, 40, 24, torch.bfloat16, seed=2)

    def grads(*which):
        ts = [t.clone().requires_grad_(n in which) for n, t in zip("xwbr", (x, w, b, r))]
        out = linear_act(ts[0], ts[1], ts[2], residual=ts[3], activation="gelu")
        out.backward(go)
        return {n: t.grad for n, t in zip("xwbr", ts)}

    full = grads(*"xwbr")
    for n in "xwbr":
        one = grads(n)
        assert torch.equal(one[n], full[n]) and all(one[m] is None for m in "xwbr" if m != n)


def test_no_rows(cuda):
    x = torch.empty(0, 16, device=cuda, requires_grad=True)
    w = torch.randn(8, 16, device=cuda, requires_grad=True)
    b = torch.randn(8, device=cuda, requires_grad=True)
    out = linear_act(x, w, b, activation="silu")
    assert out.shape == (0, 8)
    out.sum().backward()
    assert x.grad.shape == (0, 16) and (w.grad == 0).all() and (b.grad == 0).all()


def test_gradient_against_differences(cuda):
    """Directional derivatives of the operator's own outputs: a step of 1e-2 errs by about 1e-4 of the terms'
    magnitude (its square, and fp32 rounding over the step)."""
    for act in ("silu", "gelu", "none"):
        x, w, b, r, go = _make(50, 30, 20, torch.float32, seed=12)
        ts = [t.requires_grad_() for t in (x, w, b, r)]
        grads = torch.autograd.grad(linear_act(x, w, b, residual=r, activation=act), ts, go)
        for i, g in enumerate(grads):
            d = torch.randn_like(g)
            vals = []
            for sgn in (1, -1):
                moved = [t.detach() + (sgn * 1e-2 * d if j == i else 0) for j, t in enumerate(ts)]
                vals.append((linear_act(moved[0], moved[1], moved[2], residual=moved[3], activation=act).double() *
                             go.double()).sum())
            num = float(vals[0] - vals[1]) / 2e-2
            scale = float((g.double() * d).abs().sum())
            assert abs(num - float((g.double() * d).sum())) <= 1e-3 * scale + 1e-3


def test_infinities_and_nan_reach_their_own_rows_only(cuda):
    for dt in TYPES:
        x, w, b, r, go = _make(140, 80, 30, dt, seed=8)
        clean = linear_act(x, w, b, residual=r)
        x2 = x.clone()
        x2[3, 7] = float("nan")
        x2[131, 79] = float("inf")
        out = linear_act(x2, w, b, residual=r)
        keep = torch.ones(140, dtype=torch.bool, device=cuda)
        keep[3] = keep[131] = False
        assert torch.equal(out[keep], clean[keep])
        assert out[3].isnan().all() and not out[131].isfinite().any()


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 elements of the output and its gradient; x, being narrow, holds whole numbers, so that the sums
    over two million rows are exact."""
    M, K, N = 2_100_037, 8, 1032
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-1, 2, (M, K), generator=g, device=cuda).bfloat16()
    w = (torch.randint(-2, 3, (N, K), generator=g, device=cuda) / 4).bfloat16()
    xx, ww = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = linear_act(xx, ww)
    assert out.numel() > 2**31
    for rows in (slice(0, 300), slice(M - 300, M), slice(M // 2, M // 2 + 300)):
        assert torch.equal(out[rows], (x[rows].double() @ w.double().t()).bfloat16())
    go = torch.zeros(M, N, device=cuda, dtype=torch.bfloat16)
    go[-5000:] = 1
    go[:5000] = -1
    dx, dw = torch.autograd.grad(out, [xx, ww], go)
    assert torch.equal(dx[-5000:], w.double().sum(0).bfloat16().expand(5000, K)) and (dx[5000:-5000] == 0).all()
    want = x[-5000:].double().sum(0) - x[:5000].double().sum(0)
    assert torch.equal(dw, want.bfloat16().expand(N, K))


def test_other_stream_and_graph(cuda):
    x, w, b, r, go = _make(300, 64, 48, torch.bfloat16, seed=7)
    want = linear_act(x, w, b, residual=r, activation="gelu")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = linear_act(x, w, b, residual=r, activation="gelu")
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_act(x, w, b, residual=r, activation="gelu")
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_results_repeat(cuda):
    x, w, b, r, go = _make(5000, 136, 264, torch.float32, seed=11)

    def once():
        ts = [t.detach().clone().requires_grad_() for t in (x, w, b)]
        out = linear_act(*ts, activation="gelu")
        return [out.detach(), *torch.autograd.grad(out, ts, go)]

    for a, c in zip(once(), once()):
        assert torch.equal(a, c)


def test_refusals(cuda):
    x, w = torch.zeros(4, 8, device=cuda), torch.zeros(6, 8, device=cuda)
    with pytest.raises(ValueError, match="do not match"):
        linear_act(x, w[:, :7])
    with pytest.raises(TypeError):
        linear_act(x, w.half())
    with pytest.raises(ValueError, match="activation"):
        linear_act(x, w, activation="tanh")
    with pytest.raises(ValueError, match="bias"):
        linear_act(x, w, torch.zeros(5, device=cuda))
    with pytest.raises(TypeError):
        linear_act(x, w, torch.zeros(6, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="broadcast"):
        linear_act(x, w, residual=torch.zeros(3, 6, device=cuda))
    with pytest.raises(ValueError, match="empty"):
        linear_act(x, w[:0])
    with pytest.raises(ValueError, match="CUDA"):
        linear_act(x, w, torch.zeros(6))
    y = linear_act(x.requires_grad_(), w)
    g = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_no_waits_ran_out(cuda):
    torch.cuda.synchronize()
    assert _native.device_errors(clear=True) == 0
