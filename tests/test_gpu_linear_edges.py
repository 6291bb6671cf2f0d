"""linear_act where its formula, its fp32 planes or its rounding are at a limit,
against the formula in 64 bits."""

import pytest
import torch

from stockfish_trainer_b200.layer_stacks import linear_act

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
