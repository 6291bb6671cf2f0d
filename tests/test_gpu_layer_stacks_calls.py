"""How the layer-stack operators behave as calls."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from stockfish_trainer_b200.layer_stacks import block_norm, linear_act, route

pytestmark = pytest.mark.gpu


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
