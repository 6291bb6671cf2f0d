"""route against the formula in 64 bits.  Choices and counts are exact.  Gates,
loss and gradients are sums of at most 1024 exponentials held in fp32: 1e-5 of
the largest term (16-bit gradients: their unit besides)."""

import pytest
import torch

from stockfish_trainer_b200.layer_stacks import _native, route

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-9, torch.float16: 2.0**-12}
TYPES = list(UNIT)
NINF = float("-inf")


def _formula(l, k, valid, renorm):
    """Row by row, in 64 bits; returns indices, gates, counts, loss."""
    rows, E = l.shape
    idx = torch.full((rows, k), -1, dtype=torch.int64)
    counts = torch.zeros(E, dtype=torch.int64)
    gates, probs, n = [], [], 0
    for b in range(rows):
        open_ = (l[b].detach() != NINF).nonzero().flatten().tolist()
        if not open_ or (valid is not None and not valid[b]):
            gates.append(l.new_zeros(k))
            probs.append(l.new_zeros(E))
            continue
        n += 1
        p = torch.zeros_like(l[b]).index_put((torch.tensor(open_),), torch.softmax(l[b][open_], 0))
        vals = l[b].detach().tolist()
        order = sorted(open_, key=lambda e: (-vals[e], e))[:k]
        idx[b, :len(order)] = torch.tensor(order)
        for e in order:
            counts[e] += 1
        g = p[order]
        if renorm:
            g = g / g.sum()
        gates.append(torch.cat([g, l.new_zeros(k - len(order))]))
        probs.append(p)
    total = torch.stack(probs).sum(0) if rows else l.new_zeros(E)
    loss = E / (k * max(n, 1)**2) * (counts.double() * total).sum()
    return idx, torch.stack(gates) if rows else l.new_zeros(0, k), counts, loss


def _check(l, k, valid=None, renorm=True, seed=0, loss_grad=3.0):
    dt = l.dtype
    dev = l.cuda().requires_grad_()
    r = route(dev, k, valid=None if valid is None else valid.cuda(), renormalize=renorm)
    ref = l.double().requires_grad_()
    idx, gates, counts, loss = _formula(ref, k, valid, renorm)
    assert r.indices.dtype == r.counts.dtype == torch.int64 and r.gates.dtype == r.balance_loss.dtype == torch.float32
    assert torch.equal(r.indices.cpu(), idx) and torch.equal(r.counts.cpu(), counts)
    torch.testing.assert_close(r.gates.cpu().double(), gates.detach(), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(r.balance_loss.cpu().double(), loss.detach(), rtol=1e-5, atol=1e-6)
    g = torch.randn(gates.shape, generator=torch.Generator().manual_seed(seed))
    got, = torch.autograd.grad([r.gates, r.balance_loss], [dev], [g.cuda(), torch.tensor(loss_grad, device="cuda")])
    total = (gates * g.double()).sum() + loss_grad * loss
    want, = torch.autograd.grad(total, [ref]) if total.requires_grad else (torch.zeros_like(ref),)
    want = want.nan_to_num(0.0)  # the formula's own -inf entries
    assert got.dtype == dt and got.shape == l.shape
    tol = 1e-5 * (1 + want.abs().amax(1, keepdim=True)) + 2 * UNIT[dt] * want.abs() if want.numel() else want
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert (got.cpu()[l == NINF] == 0).all()


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("rows,E,k", [(1, 1, 1), (1, 8, 2), (24, 8, 1), (300, 8, 2), (77, 3, 3), (50, 16, 4),
                                      (33, 31, 5), (40, 32, 2), (41, 33, 8), (29, 67, 3), (20, 128, 6), (17, 255, 8),
                                      (9, 500, 2), (5, 1024, 40), (3, 40, 40)])
def test_sizes(cuda, rows, E, k, dt):
    g = torch.Generator().manual_seed(rows + E)
    l = (2 * torch.randn(rows, E, generator=g)).to(dt)
    for renorm in (True, False):
        _check(l, k, None, renorm)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("E,k", [(8, 2), (12, 3), (67, 5), (200, 4)])
def test_closed_experts_and_left_out_rows(cuda, E, k, dt):
    g = torch.Generator().manual_seed(E)
    l = (2 * torch.randn(120, E, generator=g)).to(dt)
    l[torch.rand(120, E, generator=g) < 0.4] = NINF
    l[5] = NINF           # nothing open
    l[6, 1:] = NINF       # one open: fewer than k
    l[7, :-1] = NINF
    l[8] = torch.finfo(dt).min  # the type's lowest value is a logit like any other: an even row
    l[9, 1:] = torch.finfo(dt).min
    valid = torch.rand(120, generator=g) < 0.8
    valid[5:10] = True
    for renorm in (True, False):
        _check(l, k, valid, renorm)
    _check(l, k, torch.zeros(120, dtype=torch.bool), True)  # no row counts
    _check(torch.full((4, E), NINF, dtype=dt), k, None, True)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_ties_go_to_the_lowest_index(cuda, dt):
    g = torch.Generator().manual_seed(1)
    l = torch.randint(-2, 3, (200, 40), generator=g).to(dt)
    l[0] = 0
    l[1, ::2] = -0.0  # equal to 0
    l[1, 1::2] = 0.0
    _check(l, 6)


def test_even_spread_has_loss_one(cuda):
    l = torch.full((64, 8), -4.0)
    l[torch.arange(64), torch.arange(64) % 8] = 0.0
    r = route(l.cuda(), 1)
    assert (r.counts == 8).all() and abs(float(r.balance_loss) - 1) < 1e-6
    same = torch.full((64, 8), -40.0)
    same[:, 3] = 0.0  # everything to one expert: the largest value, E
    assert abs(float(route(same.cuda(), 1).balance_loss) - 8) < 1e-5


def test_large_and_small_logits(cuda):
    l = torch.tensor([[3e38, -3e38, 0.0, 1.0], [1e-38, 0.0, -1e-38, -5.0], [88.0, 89.0, 90.0, -90.0]])
    _check(l, 2)
    _check(l, 3, renorm=False)


def test_nan_and_infinity(cuda):
    l = torch.randn(10, 8)
    l[2, 3] = float("nan")
    l[4] = float("nan")
    r = route(l.cuda(), 2)
    clean = torch.ones(10, dtype=torch.bool)
    clean[2] = clean[4] = False
    want = route(l[clean].cuda(), 2)
    assert torch.equal(r.indices[clean.cuda()], want.indices) and torch.equal(r.gates[clean.cuda()], want.gates)
    assert 3 not in r.indices[2].tolist() and r.gates[2].isnan().all()
    assert r.indices[4].tolist() == [-1, -1] and r.balance_loss.isnan()
    p = torch.randn(4, 8)
    p[1, 5] = float("inf")
    r = route(p.cuda(), 1)
    assert int(r.indices[1, 0]) == 5 and r.gates[1].isnan().all()


def test_many_rows(cuda):
    """Against torch on the device: enough rows for every block and several rounds."""
    g = torch.Generator(device="cuda").manual_seed(3)
    l = torch.randn(50001, 24, generator=g, device=cuda)
    valid = torch.rand(50001, generator=g, device=cuda) < 0.9
    r = route(l, 3, valid=valid)
    order = torch.argsort(l, dim=1, descending=True, stable=True)[:, :3]
    want = order.masked_fill(~valid[:, None], -1)
    assert torch.equal(r.indices, want)
    assert torch.equal(r.counts, torch.bincount(want[want >= 0], minlength=24))
    p = torch.softmax(l.double(), 1)[valid]
    n = int(valid.sum())
    loss = 24 / (3 * n * n) * (r.counts.double() * p.sum(0)).sum()
    assert abs(float(r.balance_loss) - float(loss)) < 1e-5


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 logits: the last rows' choices, gates and gradients equal those of a call on them alone."""
    rows, experts = 33_600_001, 64
    l = torch.empty(rows, experts, device=cuda, dtype=torch.bfloat16)
    l[:] = torch.randn(1, experts, device=cuda).bfloat16()
    tail = torch.randn(1000, experts, generator=torch.Generator().manual_seed(2)).bfloat16().to(cuda)
    l[-1000:] = tail
    ll = l.requires_grad_()
    r = route(ll, 1)
    want = route(tail, 1)
    assert torch.equal(r.indices[-1000:], want.indices) and torch.equal(r.gates[-1000:], want.gates)
    assert int(r.counts.sum()) == rows
    dl, = torch.autograd.grad(r.gates, ll, torch.ones_like(r.gates))
    t2 = tail.clone().requires_grad_()
    r2 = route(t2, 1)
    d2, = torch.autograd.grad(r2.gates, t2, torch.ones_like(r2.gates))
    assert torch.equal(dl[-1000:], d2)


def test_no_rows(cuda):
    l = torch.empty(0, 8, device=cuda, requires_grad=True)
    r = route(l, 2)
    assert r.indices.shape == (0, 2) and (r.counts == 0).all() and float(r.balance_loss) == 0
    (r.gates.sum() + r.balance_loss).backward()
    assert l.grad.shape == (0, 8)


def test_layouts(cuda):
    l = torch.randn(60, 12, device=cuda)
    want = route(l, 3)
    wide = torch.full((60, 20), float("nan"), device=cuda)
    wide[:, 3:15] = l
    for other in (wide[:, 3:15], l.t().contiguous().t()):
        got = route(other, 3)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    deep = route(l.view(4, 15, 12), 3, valid=torch.ones(4, 15, dtype=torch.bool, device=cuda))
    assert deep.indices.shape == (4, 15, 3) and torch.equal(deep.gates.view(60, 3), want.gates)
    one = route(l[0], 3)
    assert one.indices.shape == (3,) and torch.equal(one.indices, want.indices[0])


def test_one_output_used(cuda):
    l = torch.randn(30, 8)
    g = torch.randn(30, 2)
    for which in ("gates", "loss"):
        dev, ref = l.cuda().requires_grad_(), l.double().requires_grad_()
        r = route(dev, 2)
        _, gates, _, loss = _formula(ref, 2, None, True)
        if which == "gates":
            (r.gates * g.cuda()).sum().backward()
            (gates * g.double()).sum().backward()
        else:
            r.balance_loss.backward()
            loss.backward()
        torch.testing.assert_close(dev.grad.cpu().double(), ref.grad, rtol=1e-5, atol=1e-6)


def test_gradient_against_differences(cuda):
    """With the choices fixed, gates and loss are smooth: a step of 1e-2 on logits kept apart by more than it."""
    g = torch.Generator().manual_seed(2)
    l = (torch.stack([torch.randperm(8, generator=g) for _ in range(40)]) * 0.3).cuda().requires_grad_()
    gg = torch.randn(40, 2, generator=g).cuda()
    for renorm in (True, False):
        def value(t):
            r = route(t, 2, renormalize=renorm)
            return (r.gates.double() * gg.double()).sum() + 5 * r.balance_loss.double()

        grad, = torch.autograd.grad(value(l), l)
        d = torch.randn_like(l)
        with torch.no_grad():
            num = float(value(l + 1e-2 * d) - value(l - 1e-2 * d)) / 2e-2
        assert abs(num - float((grad * d).sum())) <= 1e-3 * float((grad * d).abs().sum()) + 1e-4


def test_results_repeat_and_graph(cuda):
    l = torch.randn(20000, 67, device=cuda)
    a, b = route(l, 3), route(l, 3)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = route(l, 3)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_refusals(cuda):
    l = torch.zeros(4, 8, device=cuda)
    for args, kw, err in (((l, 0), {}, ValueError), ((l, 9), {}, ValueError),
                          ((torch.zeros(2, 1025, device=cuda), 1), {}, ValueError),
                          ((l, 1), dict(valid=torch.ones(3, dtype=torch.bool, device=cuda)), ValueError),
                          ((l, 1), dict(valid=torch.ones(4, device=cuda)), TypeError),
                          ((l, 1), dict(valid=torch.ones(4, dtype=torch.bool)), ValueError)):
        with pytest.raises(err):
            route(*args, **kw)
    assert _native.device_errors(clear=True) == 0
