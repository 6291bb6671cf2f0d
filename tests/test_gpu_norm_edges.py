"""block_norm where a gate's meaning, its sigmoid or a call's options are at a
limit, against the formula in 64 bits."""

import threading

import pytest
import torch

from stockfish_trainer_b200.layer_stacks import _native, block_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_gates_of_a_square_input(cuda, dt):
    """As many rows as columns: a gate per row and one per column are told apart by their shape, or refused."""
    n = 48
    x, f = torch.randn(n, n, device=cuda).to(dt), torch.randn(n, n, device=cuda).to(dt)
    g = torch.rand(n, device=cuda).to(dt)
    with pytest.raises(ValueError, match="per row or per column"):
        block_norm(x, f, gate=g)
    for gate in (g[:, None], g[None, :]):
        gg = gate.clone().requires_grad_()
        y, _ = block_norm(x, f, gate=gg)
        want = x.double() + gate.double() * f.double()
        assert ((y.double() - want).abs() <= 2.0**-8 * want.abs() + 1e-6).all()
        y.sum().backward()
        dim = 1 if gate.shape[1] == 1 else 0
        err = (gg.grad.double() - f.double().sum(dim, keepdim=True)).abs()
        assert (err <= 2.0**-7 * f.double().abs().sum(dim, keepdim=True)).all()


def test_gates_whose_shape_says_enough(cuda):
    w = 5

    def y(shape, gate):
        x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).cuda()
        return block_norm(torch.zeros_like(x), x, gate=gate)[0] / x

    g = torch.rand(w, device=cuda) + 0.5
    for shape in ((w, w, w), (1, w, w), (1, 1, w, w)):
        with pytest.raises(ValueError, match="per row or per column"):
            y(shape, g.expand(shape[:-1]))
        torch.testing.assert_close(y(shape, g.expand(shape[:-1]).unsqueeze(-1)), g[:, None].expand(shape))
        torch.testing.assert_close(y(shape, g.expand(shape)), g.expand(shape))
    torch.testing.assert_close(y((3, w, w), g), g.expand(3, w, w))  # fits the columns only
    torch.testing.assert_close(y((w, 3, w), g[:, None].expand(w, 3)), g[:, None, None].expand(w, 3, w))  # the rows only
    for shape in ((1, 1), (1, 7), (1, 1, 7)):  # one row, one gate: both readings say the same
        one = torch.rand(shape[:-1], device=cuda) + 0.5
        torch.testing.assert_close(y(shape, one), one.unsqueeze(-1).expand(shape))


def test_threads_with_rows_of_different_widths(cuda):
    """One kernel asked for different amounts of shared memory by two threads at once."""
    errors = []

    def work(width):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                x = torch.randn(8, width, device=cuda)
                w = torch.ones(width, device=cuda)
                want = block_norm(x, x, post_weight=w, pre_weight=w)
                for _ in range(3000):
                    got = block_norm(x, x, post_weight=w, pre_weight=w)
                assert all(torch.equal(a, b) for a, b in zip(got, want))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(width,)) for width in (4096, 2048, 4096, 1800)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_a_gate_that_is_no_tensor_is_refused(cuda):
    x = torch.zeros(4, 8, device=cuda)
    for gate in (0.5, [1.0] * 4, torch.zeros(4)):
        with pytest.raises(TypeError if not torch.is_tensor(gate) else ValueError, match="gate"):
            block_norm(x, x, gate=gate)
    for gate in (torch.zeros(4, dtype=torch.float64, device=cuda), torch.zeros(8, dtype=torch.int64, device=cuda)):
        with pytest.raises(TypeError, match="gate"):
            block_norm(x, x, gate=gate)
    with pytest.raises(TypeError, match="gate"):  # an elementwise gate has x's type
        block_norm(x.bfloat16(), x.bfloat16(), gate=x)


def _struct(x, **kw):
    return _native.Norm(rows=x.shape[0], width=x.shape[1], dtype=_native.DTYPES[x.dtype], x=x.data_ptr(), eps=1e-5, **kw)


@pytest.mark.parametrize("width", [64, 61, 1040, 5000])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_c_forward_writes_y_without_a_block(cuda, dt, width):
    """Without f y is x, written where it is asked for."""
    x = torch.randn(9, width, device=cuda).to(dt)
    w = torch.ones(width, device=cuda)
    y, h, h2 = (torch.full_like(x, float("nan")) for _ in range(3))
    _native.run("nnue_ls_norm_forward", _struct(x, pre_weight=w.data_ptr(), y=y.data_ptr(), h=h.data_ptr()), x)
    _native.run("nnue_ls_norm_forward", _struct(x, pre_weight=w.data_ptr(), h=h2.data_ptr()), x)
    assert torch.equal(y, x) and torch.equal(h, h2) and torch.equal(h, block_norm(x, pre_weight=w)[1])
    y.fill_(0)
    _native.run("nnue_ls_norm_forward", _struct(x, y=y.data_ptr()), x)
    assert torch.equal(y, x)


@pytest.mark.parametrize("width", [64, 61, 1040, 5000])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_c_backward_without_a_block_takes_no_scale(cuda, dt, width):
    """scale_value, 0 in a zeroed struct, belongs to the block: the results are those of the Python call."""
    x = torch.randn(9, width, device=cuda).to(dt).requires_grad_()
    gh = torch.randn(9, width, device=cuda).to(dt)
    w = torch.ones(width, device=cuda)
    want, = torch.autograd.grad(block_norm(x, pre_weight=w)[1], [x], gh)
    for scale in (0.0, 1.0, 3.0):
        h, dx = torch.empty_like(x), torch.full_like(x, float("nan"))
        stats = torch.empty(9, 4, device=cuda)
        a = _struct(x, pre_weight=w.data_ptr(), h=h.data_ptr(), stats=stats.data_ptr(), scale_value=scale)
        _native.run("nnue_ls_norm_forward", a, x)
        a.grad_h, a.grad_x = gh.data_ptr(), dx.data_ptr()
        _native.run("nnue_ls_norm_backward", a, x)
        assert torch.equal(dx, want), scale


@pytest.mark.parametrize("gate", ["row", "full"])
@pytest.mark.parametrize("width", [64, 61, 5000])
def test_sigmoid_gates_far_below_zero(cuda, width, gate):
    """y = sigmoid(g) f with f alone, in relative terms: an exponential of two units, a sum, a division and two
    products; twice that for the gate's gradient (a row's is a sum of width terms of one sign)."""
    values = torch.tensor([-1.0, -10.0, -20.0, -33.0, -47.0, -60.0, -80.0], device=cuda)
    f = torch.rand(7, width, device=cuda) + 0.5
    g = (values if gate == "row" else values[:, None].expand(7, width)).clone().requires_grad_()
    y, _ = block_norm(torch.zeros_like(f), f, gate=g, gate_activation="sigmoid")
    s = torch.sigmoid(values.double())[:, None]
    assert ((y.double() - s * f.double()).abs() <= 4 * 2.0**-23 * s * f.double()).all()
    y.sum().backward()
    want = s * torch.sigmoid(-values.double())[:, None] * f.double()
    if gate == "row":
        want = want.sum(1)
    assert ((g.grad.double() - want).abs() <= 16 * 2.0**-23 * want).all(), float(((g.grad.double() - want).abs() / want).max())


@pytest.mark.parametrize("width", [64, 61, 5000])
def test_a_sum_of_squares_beyond_fp32_shows(cuda, width):
    """Values below 1.8e19 / sqrt(width) are normalised; above that the row is NaN, and no other."""
    for dt in (torch.float32, torch.bfloat16):
        x = torch.ones(3, width, device=cuda, dtype=dt)
        x[0] = 1e17
        x[1] = 3e19
        h = block_norm(x, pre_weight=torch.ones(width, device=cuda))[1]
        assert h[1].isnan().all() and ((h[[0, 2]] - 1).abs() < 1e-2).all()
