"""RoutedLayerStacks against the same network in plain torch and 64 bits, and
the example that trains it behind the feature transformer."""

import importlib.util
import os

import pytest
import torch

from stockfish_trainer_b200.layer_stacks import RoutedLayerStacks, _native

pytestmark = pytest.mark.gpu


def _rms(v, w):
    return v / torch.sqrt(v.pow(2).mean(1, keepdim=True) + 1e-5) * w


def _plain(net, p, l0, indices):
    """The network on the parameters ``p`` (64-bit copies), with the choice given."""
    silu, gelu = torch.nn.functional.silu, torch.nn.functional.gelu
    x = silu(l0 @ p["w_in"].t() + p["b_in"])
    h = _rms(x, p["first"])
    for i in range(len(net.blocks)):
        q = {k: p[f"blocks.{i}.{k}"] for k in ("w1", "b1", "w2", "b2", "gate_w", "gate_b", "post", "scale", "pre")}
        f = gelu(h @ q["w1"].t() + q["b1"]) @ q["w2"].t() + q["b2"]
        gate = torch.sigmoid(h @ q["gate_w"].t() + q["gate_b"])
        x = q["scale"] * x + gate * _rms(f, q["post"])
        h = _rms(x, q["pre"])
    logits = h @ p["w_route"].t() + p["b_route"]
    probs = torch.softmax(logits, 1)
    gates = probs.gather(1, indices)
    gates = gates / gates.sum(1, keepdim=True)
    n, e = logits.shape
    counts = torch.bincount(indices.flatten(), minlength=e).double()
    balance = e / (indices.shape[1] * n * n) * (counts * probs.sum(0)).sum()
    heads = h @ p["w_out"].t() + p["b_out"] + l0 @ p["w_skip"].t()
    return (heads.gather(1, indices) * gates).sum(1), balance, logits


@pytest.mark.parametrize("dt,tol", [(torch.float32, 2e-4), (torch.bfloat16, 0.15)])
def test_matches_plain_torch(cuda, dt, tol):
    """A dozen products and norms deep: fp32 values stay within 1e-5 of the largest, gradients (sums over the batch
    of terms that cancel) within 2e-4; in bf16 each of the dozen roundings (2^-9) adds up to a few percent."""
    torch.manual_seed(3)
    net = RoutedLayerStacks(l1=104, width=72, hidden=136, blocks=2, stacks=8, k=2)
    for name, p in net.named_parameters():
        if p.dim() == 1:
            p.data.add_(0.1 * torch.randn_like(p))
    net = net.to(cuda, dt)
    l0 = torch.rand(500, 104, device=cuda).to(dt).requires_grad_()
    value, routing = net(l0)
    target = torch.randn(500, device=cuda)
    (value * target).sum().backward()
    grads = {n: p.grad.clone() for n, p in net.named_parameters()}
    dl0 = l0.grad.clone()
    net.zero_grad()
    net(l0)[1].balance_loss.backward()
    assert net.w_route.grad.abs().max() > 0 and net.w_out.grad is None
    p = {n: q.detach().double().requires_grad_() for n, q in net.named_parameters()}
    rl0 = l0.detach().double().requires_grad_()
    want, balance, logits = _plain(net, p, rl0, routing.indices)
    chosen = logits.gather(1, routing.indices)
    assert (chosen.min(1).values >= logits.topk(2, dim=1).values[:, 1] - tol).all()  # up to rounding, the best two
    (want * target.double()).sum().backward()

    def close(a, b):
        assert (a.double() - b).norm() <= tol * b.norm() + 1e-12

    close(value.detach(), want.detach())
    assert abs(float(routing.balance_loss.detach()) - float(balance.detach())) < max(1e-5, tol * 0.1)
    close(dl0, rl0.grad)
    for n, g in grads.items():
        close(g, p[n].grad)


def test_one_position(cuda):
    net = RoutedLayerStacks(l1=1040).to(cuda)
    batch = torch.rand(40, 1040, device=cuda)
    with torch.no_grad():
        many, routes = net(batch)
        for i in (0, 7, 39):
            one, r = net(batch[i:i + 1])
            assert torch.equal(r.indices[0], routes.indices[i])
            torch.testing.assert_close(one[0], many[i], rtol=1e-4, atol=1e-5)


def test_example_trains(cuda):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "train_routed_stacks.py")
    spec = importlib.util.spec_from_file_location("train_routed_stacks", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for dt in (torch.float32, torch.bfloat16):
        losses = example.train(steps=40, batch=2048, dtype=dt, report=None)
        assert all(torch.isfinite(torch.tensor(losses))) and sum(losses[-5:]) < 0.7 * sum(losses[:5])
    assert _native.device_errors(clear=True) == 0
