"""linear_act where its formula, its fp32 planes or its rounding are at a limit,
against the formula in 64 bits."""

import math

import pytest
import torch

from stockfish_trainer_b200.layer_stacks import _native, linear_act

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12}
TYPES = list(UNIT)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("repeats,inputs", [(1, 1), (40, 1), (7, 4096)])
def test_clipped_derivatives_at_the_bounds(cuda, repeats, inputs, dt):
    """clamp passes the gradient on the closed interval, as torch's clamp and the feature transformer's epilogue do.
    A few rows, tiles, and a k range cut into pieces; every number is exact."""
    z = torch.tensor([0.0, 1.0, -0.0, 0.5, 2.0, -1.0], device=cuda, dtype=dt).repeat(repeats)
    w = torch.zeros(8, inputs, device=cuda, dtype=dt)
    w[:, 0] = 1
    for act, formula in (("relu", torch.relu), ("crelu", lambda v: v.clamp(0, 1)),
                         ("sqr_crelu", lambda v: v.clamp(0, 1) ** 2)):
        x = torch.zeros(len(z), inputs, device=cuda, dtype=dt)
        x[:, 0] = z
        x.requires_grad_()
        linear_act(x, w, activation=act).sum().backward()
        ref = z.double().requires_grad_()
        formula(ref).sum().backward()
        assert torch.equal(x.grad[:, 0].double(), 8 * ref.grad), act


@pytest.mark.parametrize("act", ["crelu", "sqr_crelu"])
def test_a_zero_layer_passes_the_gradient_that_clamp_passes(cuda, act):
    x = torch.ones(64, 16, device=cuda)
    w = torch.zeros(8, 16, device=cuda, requires_grad=True)
    linear_act(x, w, activation=act).sum().backward()
    assert (w.grad == (64 if act == "crelu" else 0)).all()


def _full_mantissas(g, *shape):
    """Values of either sign in [1, 2) whose 24 bits are all in use; some of them 0x3F80FFFF."""
    bits = 0x3F800000 | torch.randint(0, 1 << 23, shape, generator=g, dtype=torch.int32) | 1
    bits = torch.where(torch.rand(shape, generator=g) < 0.1, torch.tensor(0x3F80FFFF, dtype=torch.int32), bits)
    return bits.view(torch.float32) * (1 - 2 * torch.randint(0, 2, shape, generator=g).float())


@pytest.mark.parametrize("terms", [1, 2, 4])
def test_fp32_products_of_full_mantissas(cuda, terms):
    """Sums of `terms` products, forward, dx and dW.  What the planes leave out of a product is below 2^-24 of it and
    the sum's last add may lose a unit, 2^-23: 2^-22 of the magnitudes is allowed."""
    g = torch.Generator().manual_seed(terms)

    def check(got, a, b):
        want, mag = a.double() @ b.double().t(), a.double().abs() @ b.double().abs().t()
        err = (got.double().cpu() - want).abs() / mag
        assert err.max() <= 2.0**-22, float(err.max() * 2**23)

    x, w = _full_mantissas(g, 300, terms), _full_mantissas(g, 100, terms)
    check(linear_act(x.cuda(), w.cuda()), x, w)
    x, w, go = _full_mantissas(g, 300, 100), _full_mantissas(g, terms, 100), _full_mantissas(g, 300, terms)
    xx, ww = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dx, = torch.autograd.grad(linear_act(xx, ww), [xx], go.cuda())
    check(dx, go, w.t())
    x, w, go = _full_mantissas(g, terms, 100), _full_mantissas(g, 60, 100), _full_mantissas(g, terms, 60)
    xx, ww = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dw, = torch.autograd.grad(linear_act(xx, ww), [ww], go.cuda())
    check(dw, go.t(), x.t())


def test_fp32_values_near_the_largest(cuda):
    """Rounding a value's first plane must not make it infinite."""
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[big], [-big], [3.3961e38], [1.0]]).repeat(10, 1).cuda()
    w = torch.tensor([[1.0], [0.5], [2.0**-100 * 1.2345678], [-1.0]]).cuda()
    want = x.double() @ w.double().t()
    got = linear_act(x, w)
    assert ((got.double() - want).abs() <= 2.0**-22 * want.abs()).all()


def test_fp32_values_near_the_smallest(cuda):
    """A plane has no steps below 2^-133, so a value is held to 2^-134 or to its own rounding, whichever is more."""
    g = torch.Generator().manual_seed(1)
    scale = 10.0 ** -(30 + 8 * torch.rand(300, 40, generator=g, dtype=torch.float64))
    x = (torch.randn(300, 40, generator=g).double() * scale).float()
    w = torch.randn(24, 40, generator=g)
    want, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    err = (linear_act(x.cuda(), w.cuda()).double().cpu() - want).abs()
    tol = 2.0**-134 * w.double().abs().sum(1) + (40 / 4 + 16) * 2.0**-23 * mag + 2.0**-149
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_c_backward_of_no_rows(cuda, dt):
    """Every gradient asked for with pointers that are not null: the weight's and bias' are zero, nothing else is written."""
    code = _native.DTYPES[dt]
    dw, db, dx = (torch.full(s, float("nan"), device=cuda, dtype=dt) for s in ((24, 40), (24,), (8,)))
    a = _native.Linear(rows=0, inputs=40, outputs=24, dtype=code, bias_dtype=code, activation=4, ldg=24,
                       grad_x=dx.data_ptr(), grad_weight=dw.data_ptr(), grad_bias=db.data_ptr())
    _native.run("nnue_ls_linear_backward", a, dw)
    assert (dw == 0).all() and (db == 0).all() and dx.isnan().all()


@pytest.mark.parametrize("rows", [6, 60])
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_lower_tails_in_relative_terms(cuda, dt, rows):
    """silu and gelu far below 0, where nothing absolute would show an error.  fp32 silu: an exponential of two units,
    a sum, a division and a product.  fp32 gelu: erfc's argument is rounded, which its slope multiplies by z^2.  16-bit
    results: their own rounding, and 2^-14 for the short exponential (fp16: half its smallest step besides)."""
    u = UNIT[dt]
    for act, values in (("silu", [-5.0, -20.0, -33.0, -47.0, -60.0, -80.0]),
                        ("gelu", [-2.0, -4.0, -6.0, -8.0, -10.0, -12.0])):
        z = torch.tensor(values, device=cuda, dtype=dt).repeat(rows // 6)
        x = z[:, None].clone().requires_grad_()
        out = linear_act(x, torch.ones(1, 1, device=cuda, dtype=dt), activation=act)
        out.sum().backward()
        ref = z.double().requires_grad_()
        want = ref * torch.sigmoid(ref) if act == "silu" else ref * 0.5 * torch.special.erfc(-ref * math.sqrt(0.5))
        want.sum().backward()
        rel = 2 * u + 2.0**-14 if dt != torch.float32 else 8 * u if act == "silu" else (16 + 2 * z.double()**2) * u
        err = (out.flatten().double() - want.detach()).abs()
        assert (err <= rel * want.detach().abs() + (2.0**-25 if dt == torch.float16 else 0)).all(), (act, err / want.abs())
        if dt == torch.float32:
            err = (x.grad.flatten().double() - ref.grad).abs()
            assert (err <= 2 * rel * ref.grad.abs()).all(), (act, err / ref.grad.abs())


@pytest.fixture
def no_waiting(cuda):
    """Matrix kernels give up at once inside this: calls `on`, then `off`."""
    torch.cuda.synchronize()
    assert _native.device_errors(clear=True) == 0
    limits = []
    try:
        yield (lambda: limits.append(_native.set_wait_limit(0))), (lambda: _native.set_wait_limit(limits[0]))
    finally:
        if limits:
            _native.set_wait_limit(limits[0])
        _native.device_errors(clear=True)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("rows,inputs,outputs", [(300, 64, 48), (9, 4, 3), (40, 9000, 136), (9000, 256, 1040)])
def test_what_an_abandoned_product_leaves(no_waiting, cuda, dt, rows, inputs, outputs):
    """A wait that ran out shows in the results, forward and backward, and in the device's flags; later calls are sound."""
    on, off = no_waiting
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, go = (torch.randn(*s, generator=g, device=cuda).to(dt).requires_grad_(i < 2)
                for i, s in enumerate(((rows, inputs), (outputs, inputs), (rows, outputs))))
    b = torch.zeros(outputs, device=cuda, dtype=dt, requires_grad=True)

    def call():
        return linear_act(x, w, b, activation="silu")

    want = call()
    grads = torch.autograd.grad(want, [x, w, b], go, retain_graph=True)
    on()
    out = call()
    off()
    assert out.isnan().all() and _native.device_errors(clear=True) == _native.DEVERR_WAIT_TIMEOUT
    assert all(t.isnan().all() for t in torch.autograd.grad(out, [x, w, b], go))  # act'(z) is NaN too
    on()
    dx, dw, db = torch.autograd.grad(want, [x, w, b], go, retain_graph=True)
    off()
    assert dx.isnan().all() and dw.isnan().all() and torch.equal(db, grads[2])
    assert _native.device_errors(clear=True) == _native.DEVERR_WAIT_TIMEOUT
    again = call()
    assert torch.equal(again, want)
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(again, [x, w, b], go), grads))
    assert _native.device_errors(clear=True) == 0


def test_wait_limits(cuda):
    before = _native.set_wait_limit(7.5)
    try:
        assert before == 4 and _native.set_wait_limit(9) == 7.5
        for bad in (-1, float("nan"), float("inf")):
            with pytest.raises(ValueError):
                _native.set_wait_limit(bad)
        assert _native.set_wait_limit(before) == 9
    finally:
        _native.set_wait_limit(before)
