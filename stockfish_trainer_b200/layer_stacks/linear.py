"""Linear layer with bias, activation and residual in the product's epilogue.

The layers of the reference's stacks are separate torch calls: a product with
bias, a (squared) clamp to [0, 1], and a skip term added at the end
(src/model/modules/layer_stacks.py:15-68, stacked_linear.py:14-65).
"""

from __future__ import annotations

import torch

from . import _native

ACTIVATIONS = ("none", "relu", "crelu", "sqr_crelu", "silu", "gelu")
_ACT = {name: i for i, name in enumerate(ACTIVATIONS)}


def _args(x, weight, bias, residual, act):
    dt = _native.DTYPES[x.dtype]
    rows, inputs = x.shape
    return _native.Linear(
        rows, inputs, weight.shape[0], dt, dt if bias is None else _native.DTYPES[bias.dtype], act, 0, x.data_ptr(),
        weight.data_ptr(), None if bias is None else bias.data_ptr(), None if residual is None else residual.data_ptr(),
        max(x.stride(0), inputs), max(weight.stride(0), inputs), 0 if residual is None else _native.row_stride(residual))


def _forward(x, weight, bias, residual, act):
    a = _args(x, weight, bias, residual, act)
    out = x.new_empty((a.rows, a.outputs))
    a.out = out.data_ptr()
    _native.run("nnue_ls_linear_forward", a, x)
    return out


class LinearActFunction(torch.autograd.Function):
    """All matrices 2-D with unit column stride; bias contiguous."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        need_x, need_w = ctx.needs_input_grad[:2]
        a = _args(x, weight, bias, residual, act)
        out = x.new_empty((a.rows, a.outputs))
        a.out = out.data_ptr()
        saved, offsets = _native.linear_saved(a, 1 | 2 * need_w | 4 * need_x, x)
        _native.run("nnue_ls_linear_forward", a, x)
        # a packed form serves the backward in its original's place
        ctx.save_for_backward(x if need_w and offsets[1] < 0 else None, weight if need_x and offsets[2] < 0 else None,
                              saved)
        ctx.meta = (act, x.shape, weight.shape, x.dtype, None if bias is None else bias.dtype, offsets)
        return out

    @staticmethod
    @_native.once
    def backward(ctx, grad_out):
        x, weight, saved = ctx.saved_tensors
        act, x_shape, w_shape, dtype, bias_dtype, offsets = ctx.meta
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        grad_x = grad_w = grad_b = None
        if need_x or need_w or need_b:
            g = _native.rows_of(grad_out)
            dt = _native.DTYPES[dtype]
            a = _native.Linear(x_shape[0], x_shape[1], w_shape[0], dt,
                               dt if bias_dtype is None else _native.DTYPES[bias_dtype], act)
            if x is not None:
                a.x, a.ldx = x.data_ptr(), _native.row_stride(x)
            if weight is not None:
                a.weight, a.ldw = weight.data_ptr(), _native.row_stride(weight)
            if saved is not None:
                _native.place_saved(a, saved, offsets)
            a.grad_out, a.ldg = g.data_ptr(), _native.row_stride(g)
            if need_x:
                grad_x = g.new_empty(x_shape)
                a.grad_x = grad_x.data_ptr()
            if need_w:
                grad_w = g.new_empty(w_shape)
                a.grad_weight = grad_w.data_ptr()
            if need_b:
                grad_b = g.new_empty(w_shape[0], dtype=bias_dtype)
                a.grad_bias = grad_b.data_ptr()
            _native.run("nnue_ls_linear_backward", a, g)
        return grad_x, grad_w, grad_b, grad_out if need_r else None, None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
               residual: torch.Tensor | None = None, activation: str = "none") -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``.

    ``x`` is ``[..., inputs]`` and ``weight`` ``[outputs, inputs]``, both fp32,
    bf16 or fp16 (one type for both and for ``residual``; ``bias``
    ``[outputs]`` may also be fp32).  ``residual`` has the output's shape
    ``[..., outputs]`` or broadcasts to it.  ``activation`` is one of
    ``ACTIVATIONS``: ``crelu`` clamps to [0, 1] and ``sqr_crelu`` squares the
    result (a clamp passes gradients at its bounds too, as torch's does);
    ``gelu`` is the exact form.  Sums are held in fp32 and the result
    is rounded once; fp32 products are accurate to fp32 rounding, but with
    more than 8 rows (and in every backward) a non-finite fp32 operand may turn
    an infinite sum into NaN, and operands below 2^-110 (7.7e-34) are held to
    2^-134 instead of 24 bits.  Rows may be strided; other layouts are copied.

    For the backward ``x`` and ``weight`` (in the form their products read: for
    fp32 1.5 times their size) and the activation's derivative (as wide as the
    output) are kept; it is differentiable once.

    Should the GPU stop for longer than a product may wait for its own copies
    (4 s), what it had not formed by then is NaN, and ``device_errors()`` of
    ``layer_stacks._native`` tells it from other NaNs.
    """
    act = _ACT.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    check = _native.check_tensor
    gpu = check(x, "x")
    dt = x.dtype
    alone = _native.ALONE[dt]
    check(weight, "weight", alone, gpu)
    x_shape, w_shape = x.shape, weight.shape
    if len(x_shape) < 1 or len(w_shape) != 2 or x_shape[-1] != w_shape[1]:
        raise ValueError(f"x {tuple(x_shape)} and weight {tuple(w_shape)} do not match")
    n = w_shape[0]
    if n < 1 or w_shape[1] < 1:
        raise ValueError("weight must not be empty")
    grad = x.requires_grad or weight.requires_grad
    if bias is not None:
        check(bias, "bias", _native.OR_F32[dt], gpu)
        if bias.dim() != 1 or bias.shape[0] != n:
            raise ValueError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
        bias = bias.contiguous()
        grad = grad or bias.requires_grad
    shape = x_shape[:-1] + (n,)
    if residual is not None:
        check(residual, "residual", alone, gpu)
        if residual.shape != shape:
            try:
                residual = residual.expand(shape)
            except RuntimeError:
                raise ValueError(f"residual {tuple(residual.shape)} does not broadcast to {tuple(shape)}") from None
        residual = _native.rows_of(residual)
        grad = grad or residual.requires_grad
    x, weight = _native.rows_of(x), _native.rows_of(weight)
    if _native.differentiates(grad):
        out = LinearActFunction.apply(x, weight, bias, residual, act)
    else:
        out = _forward(x, weight, bias, residual, act)
    return out if len(shape) == 2 else out.view(shape)
