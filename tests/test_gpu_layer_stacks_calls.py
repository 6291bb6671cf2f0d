"""How the layer-stack operators behave as calls: forward-mode differentiation,
CUDA graphs of training steps, streams side by side, hooks on saved tensors."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from stockfish_trainer_b200.layer_stacks import block_norm, linear_act, route

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("call", [
    lambda x: linear_act(x, torch.ones(8, 16, device=x.device), activation="silu"),
    lambda x: linear_act(torch.zeros_like(x), torch.ones(16, 16, device=x.device), residual=x),
    lambda x: block_norm(x, pre_weight=torch.ones(16, device=x.device))[1],
    lambda x: block_norm(torch.zeros_like(x), x)[0],
    lambda x: route(x, 2).gates], ids=["linear", "residual", "norm", "block", "route"])
def test_forward_mode_is_refused(cuda, call):
    """An output without a tangent would count as a derivative of zero."""
    x = torch.randn(12, 16, device=cuda)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(call(x), call(x.clone()))  # nothing dual: an ordinary call
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))


def test_a_number_of_choices_that_is_not_whole_is_refused(cuda):
    x = torch.randn(4, 8, device=cuda)
    for k in (2.5, 2.0, "2", None):
        with pytest.raises(TypeError):
            route(x, k)
    assert route(x, True).indices.shape == (4, 1)


def _steps(dt, cuda):
    """Training steps of the three operators as functions of nothing, on tensors of their own."""
    g = torch.Generator().manual_seed(1)

    def rand(*shape, leaf=True):
        return torch.randn(*shape, generator=g).to(cuda, dt).requires_grad_(leaf)

    x, w, b, r, go = rand(300, 64), rand(48, 64), rand(48), rand(300, 48), rand(300, 48, leaf=False)
    f, p, q, gate, gy = rand(300, 64), rand(64), rand(64), rand(300, 64), rand(300, 64, leaf=False)
    l, gg = rand(300, 24), torch.randn(300, 2, generator=g).to(cuda)

    def linear():
        out = linear_act(x, w, b, residual=r, activation="gelu")
        dx, dw, db, dr = torch.autograd.grad(out, [x, w, b, r], go)
        return [out.detach(), dx, dw, db, dr.clone()]  # the residual's gradient is go itself

    def norm():
        y, h = block_norm(x, f, post_weight=p, gate=gate, gate_activation="sigmoid", pre_weight=q)
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], [x, f, p, gate, q], [gy, gy])]

    def router():
        out = route(l, 2)
        return [out.indices, out.gates.detach(), out.counts,
                *torch.autograd.grad([out.gates, out.balance_loss], [l], [gg, torch.ones((), device=cuda)])]

    return {"linear": linear, "norm": norm, "route": router}


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("name", ["linear", "norm", "route"])
def test_training_steps_in_a_graph(cuda, name, dt):
    step = _steps(dt, cuda)[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(2):
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_streams_side_by_side(cuda, dt):
    steps = _steps(dt, cuda)
    want = {n: s() for n, s in steps.items()}
    torch.cuda.synchronize()
    streams = {n: torch.cuda.Stream() for n in steps}
    got = {n: [] for n in steps}
    for _ in range(20):
        for n, s in steps.items():
            with torch.cuda.stream(streams[n]):
                got[n].append(s())
    torch.cuda.synchronize()
    for n in steps:
        for again in got[n]:
            assert all(torch.equal(a, b) for a, b in zip(again, want[n])), n


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_saved_tensor_hooks(cuda, dt):
    """What the forward keeps may wait elsewhere; strided rows come back contiguous."""
    for n, step in _steps(dt, cuda).items():
        want = step()
        with torch.autograd.graph.save_on_cpu():
            assert all(torch.equal(a, b) for a, b in zip(step(), want)), n
    wide = torch.randn(40, 72, device=cuda).to(dt)
    w = torch.randn(12, 63, device=cuda).to(dt).requires_grad_()
    go = torch.randn(40, 12, device=cuda).to(dt)

    def strided():
        x = wide[:, :63].detach().requires_grad_()
        return torch.autograd.grad(linear_act(x, w, activation="silu"), [x, w], go)

    want = strided()
    with torch.autograd.graph.save_on_cpu():
        got = strided()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
