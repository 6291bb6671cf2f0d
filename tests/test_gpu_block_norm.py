"""block_norm against the formula in 64 bits.

Tolerances.  Statistics and sums in fp32 over `width` (up to a few thousand)
terms added in trees, and a dozen further operations, stay within 2^-24 * 64
(4e-6) of the largest term that enters a row's result; so fp32 outputs may be
off by 1e-5 of their row's largest term, 16-bit ones by their unit besides.
Sums over rows may be off by 1e-5 of the sum of their terms' magnitudes."""

import pytest
import torch

from stockfish_trainer_b200.layer_stacks import block_norm

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12}
TYPES = list(UNIT)
EPS = 1e-5


def _norm(v, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS)


def _formula(t, kind, sigmoid, scale_value=1.0):
    """(y, h) of a dict of tensors, in their own precision."""
    y = t["x"]
    if t.get("f") is not None:
        n = t["f"]
        if t.get("post_weight") is not None:
            n = _norm(n, kind) * t["post_weight"]
            if t.get("post_bias") is not None:
                n = n + t["post_bias"]
        if t.get("gate") is not None:
            g = torch.sigmoid(t["gate"]) if sigmoid else t["gate"]
            n = n * (g.unsqueeze(-1) if g.dim() == y.dim() - 1 else g)
        s = t["residual_scale"] if t.get("residual_scale") is not None else scale_value
        y = s * y + n
    h = None
    if t.get("pre_weight") is not None:
        h = _norm(y, kind) * t["pre_weight"]
        if t.get("pre_bias") is not None:
            h = h + t["pre_bias"]
    return y, h


def _make(rows, width, dt, seed, gate="none", learned=True, bias=True, f=True, post=True, pre=True, params=None,
          gate_dt=None):
    g = torch.Generator().manual_seed(seed)
    params = params or torch.float32
    t = {"x": torch.randn(rows, width, generator=g).to(dt)}
    if f:
        t["f"] = (2 * torch.randn(rows, width, generator=g) + 0.5).to(dt)
        if post:
            t["post_weight"] = (1 + 0.2 * torch.randn(width, generator=g)).to(params)
            if bias:
                t["post_bias"] = (0.2 * torch.randn(width, generator=g)).to(params)
        if learned:
            t["residual_scale"] = (0.9 + 0.1 * torch.randn(width, generator=g)).to(params)
        if gate == "row":
            t["gate"] = (torch.rand(rows, generator=g) + 0.1).to(gate_dt or torch.float32)
        elif gate == "full":
            t["gate"] = torch.randn(rows, width, generator=g).to(dt)
    if pre:
        t["pre_weight"] = (1 + 0.2 * torch.randn(width, generator=g)).to(params)
        if bias:
            t["pre_bias"] = (0.2 * torch.randn(width, generator=g)).to(params)
    return t, torch.randn(rows, width, generator=g).to(dt), torch.randn(rows, width, generator=g).to(dt)


def _call(t, kind, sigmoid, scale_value=1.0):
    kw = {k: v for k, v in t.items() if k not in ("x", "f")}
    kw.setdefault("residual_scale", scale_value)
    return block_norm(t["x"], t.get("f"), gate_activation="sigmoid" if sigmoid else "none", kind=kind, eps=EPS, **kw)


def _check(t, gy, gh, kind, sigmoid=False, scale_value=1.0):
    dt = t["x"].dtype
    u = UNIT[dt]
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    ref = {k: v.double().requires_grad_() for k, v in t.items()}
    y, h = _call(dev, kind, sigmoid, scale_value)
    ry, rh = _formula(ref, kind, sigmoid, scale_value)
    outs, routs, grads = [], [], []
    for have, want, grad in ((y, ry, gy), (h, rh, gh)):
        assert (have is None) == (want is None)
        if have is None:
            continue
        assert have.dtype == dt and have.shape == want.shape
        err = (have.detach().double().cpu() - want.detach()).abs()
        top = want.detach().abs().amax(1, keepdim=True) + 1
        assert (err <= 1e-5 * top + 2 * u * want.detach().abs()).all(), float((err / top).max())
        if have.requires_grad and have is not dev["x"]:
            outs.append(have)
            routs.append(want)
            grads.append(grad)
    got = torch.autograd.grad(outs, list(dev.values()), [g.cuda() for g in grads])
    want = torch.autograd.grad(routs, list(ref.values()), [g.double() for g in grads], retain_graph=True)
    # per-row terms of the sums over rows: the same gradients with the parameter spread over the rows
    spread = {k: (v.detach().expand(t["x"].shape).clone().requires_grad_() if v.dim() == 1 and k != "gate" else v)
              for k, v in ref.items()}
    sy, sh = _formula(spread, kind, sigmoid, scale_value)
    souts = [o for o in (sy, sh) if o is not None]
    if t.get("f") is None:
        souts = [sh]
    terms = torch.autograd.grad(souts, list(spread.values()), [g.double() for g in grads])
    for name, a, b, s in zip(t, got, want, terms):
        assert a.dtype == t[name].dtype and a.shape == b.shape, name
        err = (a.double().cpu() - b).abs()
        if a.dim() == 2:
            tol = 1e-5 * (b.abs().amax(1, keepdim=True) + 1e-2) * 4 + 2 * u * b.abs()
        elif name == "gate":  # a sum over the row's width, whose terms are of the order of grad_y and grad_h
            tol = 1e-5 * t["x"].shape[1] * 8 + 2 * UNIT[a.dtype] * b.abs()
        else:
            tol = 1e-5 * 4 * (s.abs().sum(0) + 1e-2) + 2 * UNIT[a.dtype] * b.abs()
        tol = tol + (6e-8 if a.dtype == torch.float16 else 0)
        assert (err <= tol).all(), (name, float((err / tol).max()))


SIZES = [(1, 1), (1, 1040), (2, 7), (5, 16), (37, 128), (300, 1031), (64, 1048), (700, 520), (11, 2050), (9, 4096),
         (3, 9001), (2, 20000)]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", SIZES)
def test_sizes(cuda, rows, width, kind, dt):
    gate = ["none", "row", "full"][(rows + width) % 3]
    t, gy, gh = _make(rows, width, dt, rows * 31 + width, gate=gate)
    if width == 1 and kind == "layer":
        # the norm of one value is 0 whatever it is; its gradients are 0 * 1/sqrt(eps), not a test of sums
        y, h = _call({k: v.cuda() for k, v in t.items()}, kind, False)
        assert torch.equal(h.cpu().float(), t["pre_bias"].expand(rows, 1).to(dt).float())
        return
    _check(t, gy, gh, kind)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("gate", ["none", "row", "full"])
@pytest.mark.parametrize("rows,width", [(900, 1152), (700, 1156), (333, 1536), (5, 2048), (1000, 1160), (40, 2044),
                                        (400, 2052), (301, 4096), (333, 4095), (7, 4100)])
def test_widths_around_the_kernels_limits(cuda, rows, width, gate, dt):
    for kind in ("rms", "layer"):
        t, gy, gh = _make(rows, width, dt, rows + width, gate=gate)
        _check(t, gy, gh, kind, sigmoid=True)


@pytest.mark.parametrize("gate", ["none", "row", "full"])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("learned", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("width", [96, 133])
def test_forms(cuda, gate, sigmoid, learned, bias, width):
    for kind in ("rms", "layer"):
        t, gy, gh = _make(50, width, torch.float32, 17, gate=gate, learned=learned, bias=bias)
        _check(t, gy, gh, kind, sigmoid, scale_value=0.75)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("f,post,pre", [(False, False, True), (True, False, True), (True, True, False),
                                        (True, False, False)])
def test_parts(cuda, f, post, pre, dt):
    """Only the norm before, only the norm after, neither."""
    t, gy, gh = _make(40, 264, dt, 23, gate="row" if f else "none", learned=False, f=f, post=post, pre=pre)
    gys = gy if f else gh
    for kind in ("rms", "layer"):
        _check(t, gys, gh, kind)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
def test_types_of_parameters_and_gate(cuda, dt):
    for params, gate_dt in ((dt, dt), (dt, torch.float32), (torch.float32, dt)):
        t, gy, gh = _make(33, 72, dt, 29, gate="row", params=params, gate_dt=gate_dt)
        _check(t, gy, gh, "rms", sigmoid=True)


def test_large_offset_keeps_the_variance(cuda):
    """Layer norm of values around 1000: the variance is formed from differences to the mean."""
    t, gy, gh = _make(20, 1040, torch.float32, 31, gate="none", learned=False)
    t["f"] = t["f"] + 1000
    y, h = _call({k: v.cuda() for k, v in t.items()}, "layer", False)
    ry, rh = _formula({k: v.double() for k, v in t.items()}, "layer", False)
    # the mean of values near 1000 is known to 2^-24 * 1000 * a few = 3e-4 of the values' spread
    assert (y.double().cpu() - ry).abs().max() < 2e-3 and (h.double().cpu() - rh).abs().max() < 2e-3


def test_zero_rows_and_zero_values(cuda):
    t, gy, gh = _make(6, 40, torch.float32, 1, gate="row")
    t["f"][2] = 0
    t["x"][2] = 0
    _check(t, gy * 0.01, gh * 0.01, "rms")
    e, gy, gh = _make(0, 40, torch.float32, 1, gate="row")
    dev = {k: v.cuda().requires_grad_() for k, v in e.items()}
    y, h = _call(dev, "rms", False)
    assert y.shape == h.shape == (0, 40)
    for g in torch.autograd.grad([y, h], list(dev.values()), [gy.cuda(), gh.cuda()]):
        assert g.numel() == 0 or (g == 0).all()


def test_one_output_used(cuda):
    t, gy, gh = _make(30, 136, torch.bfloat16, 3, gate="full")
    for which in (0, 1):
        dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
        ref = {k: v.double().requires_grad_() for k, v in t.items()}
        used = {k: v for k, v in dev.items() if which == 1 or not k.startswith("pre_")}
        got = torch.autograd.grad(_call(dev, "rms", True)[which], list(used.values()), (gy, gh)[which].cuda())
        want = torch.autograd.grad(_formula(ref, "rms", True)[which], [ref[k] for k in used], (gy, gh)[which].double())
        for name, a, b in zip(used, got, want):
            err = (a.double().cpu() - b).abs()
            assert (err <= 2 * UNIT[a.dtype] * b.abs() + 1e-4).all(), name


def test_layouts(cuda):
    t, gy, gh = _make(60, 88, torch.float32, 5, gate="full")
    dev = {k: v.cuda() for k, v in t.items()}
    y, h = _call(dev, "layer", True)
    buf = torch.zeros(60 * 88 + 1, device=cuda)  # breaks 16-byte alignment
    off = dict(dev, x=buf[1:].view(60, 88).copy_(dev["x"]))
    y2, h2 = _call(off, "layer", True)
    torch.testing.assert_close(y2, y, rtol=1e-6, atol=1e-6)
    torch.testing.assert_close(h2, h, rtol=1e-5, atol=1e-5)
    tr = dict(dev, f=dev["f"].t().contiguous().t())
    assert torch.equal(_call(tr, "layer", True)[0], y)
    deep = {k: v.view(3, 20, 88) if v.dim() == 2 else v for k, v in dev.items()}
    y3, h3 = _call(deep, "layer", True)
    assert y3.shape == (3, 20, 88) and torch.equal(y3.view(60, 88), y) and torch.equal(h3.view(60, 88), h)
    row = torch.rand(3, 20, 1, device=cuda, requires_grad=True)
    y4, _ = block_norm(deep["x"], deep["f"], gate=row)
    y4.sum().backward()
    assert row.grad.shape == row.shape
    torch.testing.assert_close(row.grad, deep["f"].sum(-1, keepdim=True), rtol=1e-4, atol=1e-4)
    col = torch.rand(88, device=cuda, requires_grad=True)  # one gate per column: broadcast, its gradient summed
    y5, _ = block_norm(dev["x"], dev["f"], gate=col)
    y5.sum().backward()
    torch.testing.assert_close(col.grad, dev["f"].sum(0), rtol=1e-4, atol=1e-4)


def test_gradient_against_differences(cuda):
    """A step of 1e-2 errs by its square against the terms' magnitude, and by fp32 rounding over the step."""
    for kind in ("rms", "layer"):
        t, gy, gh = _make(40, 64, torch.float32, 41, gate="full")
        dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
        y, h = _call(dev, kind, True)
        grads = torch.autograd.grad([y, h], list(dev.values()), [gy.cuda(), gh.cuda()])
        for name, g in zip(dev, grads):
            d = torch.randn_like(g)
            vals = []
            for sgn in (1, -1):
                moved = {k: (v + sgn * 1e-2 * d if k == name else v).detach() for k, v in dev.items()}
                a, b = _call(moved, kind, True)
                vals.append((a.double() * gy.cuda().double()).sum() + (b.double() * gh.cuda().double()).sum())
            num, ana = float(vals[0] - vals[1]) / 2e-2, float((g.double() * d).sum())
            assert abs(num - ana) <= 2e-3 * float((g.double() * d).abs().sum()) + 1e-3, name


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 elements: the last rows equal those of a call on them alone, bit for bit."""
    rows, width = 2_100_037, 1032
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, width, generator=g, device=cuda, dtype=torch.bfloat16)
    f = torch.randn(rows, width, generator=g, device=cuda, dtype=torch.bfloat16)
    w = torch.rand(width, device=cuda) + 0.5
    y, h = block_norm(x, f, post_weight=w, pre_weight=w)
    for part in (slice(rows - 64, rows), slice(0, 64)):
        y2, h2 = block_norm(x[part], f[part], post_weight=w, pre_weight=w)
        assert torch.equal(y[part], y2) and torch.equal(h[part], h2)
    del y, h
    xx, ff = x.requires_grad_(), f.requires_grad_()
    out = block_norm(xx, ff, post_weight=w, pre_weight=w)[1]
    dx, df = torch.autograd.grad(out, [xx, ff], out.detach())
    part = slice(rows - 64, rows)
    xs, fs = x[part].detach().requires_grad_(), f[part].detach().requires_grad_()
    o2 = block_norm(xs, fs, post_weight=w, pre_weight=w)[1]
    for a, b in zip((dx, df), torch.autograd.grad(o2, [xs, fs], out[part].detach())):
        assert torch.equal(a[part], b)


def test_nan_stays_in_its_row(cuda):
    t, gy, gh = _make(20, 136, torch.bfloat16, 7, gate="row")
    dev = {k: v.cuda() for k, v in t.items()}
    y, h = _call(dev, "rms", False)
    dev["f"][4, 3] = float("nan")
    dev["x"][9, 0] = float("inf")
    y2, h2 = _call(dev, "rms", False)
    keep = [i for i in range(20) if i not in (4, 9)]
    assert torch.equal(y2[keep], y[keep]) and torch.equal(h2[keep], h[keep])
    assert y2[4].isnan().all() and h2[4].isnan().all() and h2[9].isnan().any()


def test_results_repeat(cuda):
    t, gy, gh = _make(3000, 264, torch.bfloat16, 9, gate="row")

    def once():
        dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
        y, h = _call(dev, "layer", False)
        return [y, h, *torch.autograd.grad([y, h], list(dev.values()), [gy.cuda(), gh.cuda()])]

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_refusals(cuda):
    x, w = torch.zeros(4, 8, device=cuda), torch.ones(8, device=cuda)
    for kw, err in ((dict(), ValueError), (dict(pre_weight=w[:7]), ValueError), (dict(pre_weight=w.half()), TypeError),
                    (dict(pre_weight=w, kind="batch"), ValueError), (dict(pre_weight=w, eps=-1.0), ValueError),
                    (dict(pre_weight=w, gate=w), ValueError), (dict(pre_bias=w), ValueError),
                    (dict(pre_weight=w, residual_scale=2.0), ValueError),
                    (dict(f=x[:3], pre_weight=w), ValueError), (dict(f=x.half()), TypeError),
                    (dict(f=x, post_bias=w), ValueError), (dict(f=x, gate=torch.zeros(3, device=cuda)), ValueError),
                    (dict(f=x, gate_activation="tanh"), ValueError), (dict(f=x, post_weight=w.cpu()), ValueError),
                    (dict(f=x.bfloat16()), TypeError)):
        with pytest.raises(err):
            block_norm(x, **kw)
    xb = x.bfloat16()
    with pytest.raises(TypeError):  # parameters share one type
        block_norm(xb, xb, post_weight=w, pre_weight=w.bfloat16())


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 3), (2, 7), (5, 33), (700, 129), (9, 1031), (3, 4095)])
def test_rows_from_any_byte(cuda, dt, rows, width):
    # where the tensors start changes nothing, not even the rounding
    t, gy, gh = _make(rows, width, dt, 6, gate="full")
    wants = None
    for offset in (0, 1, 3, 5):
        def place(v, offset=offset):
            if v.dim() == 1:
                return v.cuda()
            return torch.full((v.numel() + offset,), float("nan"), dtype=dt, device="cuda")[offset:].view(v.shape).copy_(v)
        dev = {k: place(v).requires_grad_() for k, v in t.items()}
        outs = _call(dev, "layer", True)
        got = [*outs, *torch.autograd.grad(outs, list(dev.values()), [place(gy), place(gh)])]
        wants = wants or got
        assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(got, wants))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [k * 256 - d for k in range(1, 17) for d in (0, 1)])
def test_every_block_size(cuda, dt, width):
    # each width of a block asks for its own amount of shared memory, with and without the optional terms
    for gate, more in (("row", False), ("full", False), ("row", True), ("full", True)):
        t, gy, gh = _make(5, width, dt, 7, gate=gate, learned=more, bias=more)
        _check(t, gy, gh, "layer", True)
