"""Router of the layer stacks: which experts a position goes to, how often each
was chosen, and the balance loss that keeps the choice spread.

The reference's router picks its stacks in torch (src/model/modules/
moe_stacks.py:12-283)."""

from __future__ import annotations

import operator
from typing import NamedTuple

import torch

from . import _native


class Routing(NamedTuple):
    """``indices`` [..., k] int64 (-1 = no choice), ``gates`` [..., k] fp32,
    ``counts`` [experts] int64, ``balance_loss`` fp32 scalar."""

    indices: torch.Tensor
    gates: torch.Tensor
    counts: torch.Tensor
    balance_loss: torch.Tensor


def _args(logits, valid, k, renormalize, indices, gates, counts, loss):
    rows, experts = logits.shape
    return _native.Route(rows, experts, k, _native.DTYPES[logits.dtype], renormalize, logits.data_ptr(),
                         max(logits.stride(0), experts), None if valid is None else valid.data_ptr(),
                         indices.data_ptr(), gates.data_ptr(), counts.data_ptr(), loss.data_ptr())


def _forward(logits, valid, k, renormalize):
    rows, experts = logits.shape
    indices = logits.new_empty((rows, k), dtype=torch.int64)
    gates = logits.new_empty((rows, k), dtype=torch.float32)
    counts = logits.new_empty(experts, dtype=torch.int64)
    loss = logits.new_empty(2, dtype=torch.float32)
    _native.run("nnue_ls_route_forward", _args(logits, valid, k, renormalize, indices, gates, counts, loss), logits)
    return indices, gates, counts, loss


class RouteFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, valid, k, renormalize):
        indices, gates, counts, loss = _forward(logits, valid, k, renormalize)
        ctx.save_for_backward(logits, valid, indices, gates, counts, loss)
        ctx.meta = (k, renormalize)
        ctx.mark_non_differentiable(indices, counts)
        ctx.set_materialize_grads(False)
        return indices, gates, counts, loss[0]

    @staticmethod
    @_native.once
    def backward(ctx, _indices, grad_gates, _counts, grad_loss):
        logits, valid, indices, gates, counts, loss = ctx.saved_tensors
        a = _args(logits, valid, *ctx.meta, indices, gates, counts, loss)
        if grad_gates is not None:
            grad_gates = grad_gates.contiguous()
            a.grad_gates = grad_gates.data_ptr()
        if grad_loss is not None:
            grad_loss = grad_loss.contiguous()
            a.grad_loss = grad_loss.data_ptr()
        grad = logits.new_empty(logits.shape)
        a.grad_logits = grad.data_ptr()
        _native.run("nnue_ls_route_backward", a, logits)
        return grad, None, None, None


def route(logits: torch.Tensor, k: int, *, valid: torch.Tensor | None = None, renormalize: bool = True) -> Routing:
    """Choose ``k`` experts per row of ``logits`` ``[..., experts]`` (fp32, bf16
    or fp16), count the choices and form the balance loss.

    With p = softmax(logits) a row's choices are its k largest logits, largest
    first, ties to the lowest index; their gates are p there, divided by their
    sum with ``renormalize``.  Over the n rows that count::

        balance_loss = experts / (k n^2) * sum_e counts[e] * sum_rows p[row, e]

    which is 1 when choices and probabilities are spread evenly.  A row counts
    if ``valid`` (bool ``[...]``, default all) says so and it has a logit other
    than -inf; an expert at -inf is closed to the row.  Rows that do not count,
    and choices beyond the open experts, have index -1 and gate 0, and get no
    gradient.  A NaN logit is never chosen and makes the gates of its row's
    choices and the loss NaN.  ``gates`` and ``balance_loss`` carry gradients to ``logits``;
    the counts enter them as constants.  Probabilities, gates and sums are held
    in fp32.
    """
    gpu = _native.check_tensor(logits, "logits")
    shape = logits.shape
    if len(shape) < 1 or not 1 <= shape[-1] <= _native.MAX_EXPERTS:
        raise ValueError(f"logits must be [..., experts] with 1 <= experts <= {_native.MAX_EXPERTS}, "
                         f"got {tuple(shape)}")
    k = operator.index(k)
    if not 1 <= k <= shape[-1]:
        raise ValueError(f"k must be in [1, {shape[-1]}], got {k}")
    shape = shape[:-1]
    if valid is not None:
        _native.check_tensor(valid, "valid", (torch.bool,), gpu)
        if valid.shape != shape:
            raise ValueError(f"valid must have shape {tuple(shape)}, got {tuple(valid.shape)}")
        valid = valid.reshape(-1).contiguous()
    rows = _native.rows_of(logits)
    if _native.differentiates(logits.requires_grad):
        indices, gates, counts, loss = RouteFunction.apply(rows, valid, k, bool(renormalize))
    else:
        indices, gates, counts, loss = _forward(rows, valid, k, bool(renormalize))
        loss = loss[0]
    if len(shape) != 1:
        indices, gates = indices.view(*shape, k), gates.view(*shape, k)
    return Routing(indices, gates, counts, loss)
