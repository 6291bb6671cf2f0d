"""Operators of the dense layers behind the feature transformer (reference
src/model/modules/layer_stacks.py, stacked_linear.py, moe_stacks.py), forward
and backward as hand-written kernels (include/nnue_ls.h):

* ``linear_act``  out = act(x W^T + b) + residual;
* ``block_norm``  the norms before and after a residual block, with the block's
  gate and residual scale;
* ``route``       a router's top-k choice with per-expert counts and the balance
  loss.

They are differentiable once, in reverse mode; forward mode is refused.

``RoutedLayerStacks`` puts them together.
"""

from .linear import ACTIVATIONS, linear_act
from .norm import block_norm
from .router import Routing, route
from .stacks import ResidualBlock, RoutedLayerStacks

__all__ = ["ACTIVATIONS", "linear_act", "block_norm", "route", "Routing", "ResidualBlock", "RoutedLayerStacks"]
