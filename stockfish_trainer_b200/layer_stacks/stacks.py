"""The dense part of the network behind the feature transformer, built from the
operators of this package: a trunk of gated residual blocks, a value head per
stack and a router that mixes them.

Like the reference's stacks (src/model/modules/layer_stacks.py:15-68) it takes
``l0`` from ``transform_inputs`` and adds a direct product of ``l0`` to each
stack's output; like its routed form (src/model/modules/moe_stacks.py:12-283)
it computes every stack for every position and mixes the chosen ones.
"""

from __future__ import annotations

import math

import torch
from torch import nn

from .linear import linear_act
from .norm import block_norm
from .router import Routing, route


def _weight(outputs: int, inputs: int, scale: float = 1.0) -> nn.Parameter:
    bound = scale / math.sqrt(inputs)
    return nn.Parameter(torch.empty(outputs, inputs).uniform_(-bound, bound))


class ResidualBlock(nn.Module):
    """``f(h) = W2 gelu(W1 h + b1) + b2``, its per-position gate, and the norms
    that close it and open what follows."""

    def __init__(self, width: int, hidden: int):
        super().__init__()
        self.w1, self.b1 = _weight(hidden, width), nn.Parameter(torch.zeros(hidden))
        self.w2, self.b2 = _weight(width, hidden), nn.Parameter(torch.zeros(width))
        self.gate_w, self.gate_b = _weight(1, width), nn.Parameter(torch.zeros(1))
        self.post = nn.Parameter(torch.ones(width))
        self.scale = nn.Parameter(torch.ones(width))
        self.pre = nn.Parameter(torch.ones(width))

    def forward(self, x: torch.Tensor, h: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        f = linear_act(linear_act(h, self.w1, self.b1, activation="gelu"), self.w2, self.b2)
        gate = linear_act(h, self.gate_w, self.gate_b)
        return block_norm(x, f, post_weight=self.post, gate=gate, gate_activation="sigmoid", residual_scale=self.scale,
                          pre_weight=self.pre)


class RoutedLayerStacks(nn.Module):
    """``forward(l0, valid=None) -> (value [B], Routing)``.

    ``l1`` is the feature transformer's width, ``stacks`` the number of value
    heads of which ``k`` are mixed per position.  Add ``Routing.balance_loss``,
    weighted, to the training loss.  ``.to(torch.bfloat16)`` runs the trunk in
    16 bits; the gates of the mixture stay in 32.
    """

    def __init__(self, l1: int = 1040, width: int = 256, hidden: int = 512, blocks: int = 2, stacks: int = 8, k: int = 2):
        super().__init__()
        self.k = k
        self.w_in, self.b_in = _weight(width, l1), nn.Parameter(torch.zeros(width))
        self.first = nn.Parameter(torch.ones(width))
        self.blocks = nn.ModuleList(ResidualBlock(width, hidden) for _ in range(blocks))
        self.w_route, self.b_route = _weight(stacks, width), nn.Parameter(torch.zeros(stacks))
        self.w_skip = _weight(stacks, l1)
        self.w_out, self.b_out = _weight(stacks, width), nn.Parameter(torch.zeros(stacks))

    def forward(self, l0: torch.Tensor, valid: torch.Tensor | None = None) -> tuple[torch.Tensor, Routing]:
        x = linear_act(l0, self.w_in, self.b_in, activation="silu")
        x, h = block_norm(x, pre_weight=self.first)
        for block in self.blocks:
            x, h = block(x, h)
        routing = route(linear_act(h, self.w_route, self.b_route), self.k, valid=valid)
        heads = linear_act(h, self.w_out, self.b_out, residual=linear_act(l0, self.w_skip))
        chosen = heads.gather(1, routing.indices.clamp_min(0)).float()
        return (chosen * routing.gates).sum(1), routing
