"""Norms before and after a residual block, fused with the block's gate and
residual scale, as one kernel each way."""

from __future__ import annotations

import torch

from . import _native

_KINDS = {"rms": 0, "layer": 1}
_PARAMS = ("post_weight", "post_bias", "residual_scale", "pre_weight", "pre_bias")


def _args(x, f, gate, params, meta):
    dt = _native.DTYPES[x.dtype]
    kind, gate_mode, gate_sigmoid, scale_value, eps, params_dtype, gate_dtype = meta
    rows, width = x.shape
    return _native.Norm(rows, width, dt, params_dtype, gate_dtype, kind, gate_mode, gate_sigmoid, scale_value, eps, 0,
                        x.data_ptr(), None if f is None else f.data_ptr(), None if gate is None else gate.data_ptr(),
                        *[None if t is None else t.data_ptr() for t in params])


def _forward(x, f, gate, params, meta, want_stats):
    a = _args(x, f, gate, params, meta)
    y = h = stats = None
    if f is not None:
        y = torch.empty_like(x)
        a.y = y.data_ptr()
    if params[3] is not None:
        h = torch.empty_like(x)
        a.h = h.data_ptr()
    if want_stats:
        stats = x.new_empty((x.shape[0], 4), dtype=torch.float32)
        a.stats = stats.data_ptr()
    _native.run("nnue_ls_norm_forward", a, x)
    return y, h, stats


class BlockNormFunction(torch.autograd.Function):
    """Returns (y, h); without ``f`` y is ``None`` (it is x), without
    ``pre_weight`` h is ``None``.  All tensors contiguous, x and f 2-D."""

    @staticmethod
    def forward(ctx, x, f, gate, post_weight, post_bias, scale, pre_weight, pre_bias, meta):
        params = (post_weight, post_bias, scale, pre_weight, pre_bias)
        y, h, stats = _forward(x, f, gate, params, meta, True)
        ctx.save_for_backward(x, f, gate, stats, *params)
        ctx.meta = meta
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @_native.once
    def backward(ctx, grad_y, grad_h):
        x, f, gate, stats, *params = ctx.saved_tensors
        need = ctx.needs_input_grad
        a = _args(x, f, gate, params, ctx.meta)
        a.stats = stats.data_ptr()
        if grad_y is not None:
            grad_y = grad_y.contiguous()
            a.grad_y = grad_y.data_ptr()
        if grad_h is not None:
            grad_h = grad_h.contiguous()
            a.grad_h = grad_h.data_ptr()
        grads = [torch.empty_like(t) if n and t is not None else None for n, t in zip(need, (x, f, gate, *params))]
        (a.grad_x, a.grad_f, a.grad_gate, a.grad_post_weight, a.grad_post_bias, a.grad_scale, a.grad_pre_weight,
         a.grad_pre_bias) = [None if g is None else g.data_ptr() for g in grads]
        _native.run("nnue_ls_norm_backward", a, x)
        return (*grads, None)


def block_norm(x: torch.Tensor, f: torch.Tensor | None = None, *, post_weight: torch.Tensor | None = None,
               post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None, gate_activation: str = "none",
               residual_scale: float | torch.Tensor = 1.0, pre_weight: torch.Tensor | None = None,
               pre_bias: torch.Tensor | None = None, kind: str = "rms",
               eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Close one residual block and open the next::

        n = norm(f) * post_weight + post_bias      # n = f without post_weight
        y = residual_scale * x + gate * n          # y = x without f
        h = norm(y) * pre_weight + pre_bias        # h is None without pre_weight

    and return ``(y, h)``.  ``x`` (the residual stream) and ``f`` (the block's
    output) are ``[..., width]`` in fp32, bf16 or fp16; ``norm`` is the
    ``"rms"`` or ``"layer"`` norm of a row.  ``gate`` is one value per row
    (``[...]`` or ``[..., 1]``, also in fp32), or elementwise (broadcast to
    x's shape, in x's type); a shape that says both, such as ``[n]`` beside
    ``[n, n]``, is refused: give it as ``[n, 1]`` or ``[1, n]``.  With
    ``gate_activation="sigmoid"`` the gate goes through a sigmoid first.
    ``residual_scale`` is a number or a learned ``[width]`` tensor.  The
    parameters share one type, x's or fp32.  Statistics and sums are held in
    fp32 (a row whose squares sum past its range, with values from 1.8e19 /
    sqrt(width) up, becomes NaN), h is normalised from the unrounded y, and each
    output is rounded once.  Differentiable once, in every tensor argument.
    """
    check = _native.check_tensor
    gpu = check(x, "x")
    dt = x.dtype
    alone, mixed = _native.ALONE[dt], _native.OR_F32[dt]
    if kind not in _KINDS:
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    if gate_activation not in ("none", "sigmoid"):
        raise ValueError(f"gate_activation must be 'none' or 'sigmoid', got {gate_activation!r}")
    shape = x.shape
    if len(shape) < 1 or not 1 <= shape[-1] <= _native.NORM_MAX_WIDTH:
        raise ValueError(f"x must be [..., width] with 1 <= width <= {_native.NORM_MAX_WIDTH}, got {tuple(shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    width = shape[-1]
    grad = x.requires_grad
    scale, scale_value = None, 1.0
    if isinstance(residual_scale, torch.Tensor):
        scale = residual_scale
    else:
        scale_value = float(residual_scale)
    if f is None:
        if post_weight is not None or gate is not None or scale is not None or scale_value != 1.0:
            raise ValueError("post_weight, gate and residual_scale belong to a block's output f")
        if pre_weight is None:
            raise ValueError("nothing to do: give f, pre_weight or both")
    else:
        check(f, "f", alone, gpu)
        if f.shape != shape:
            raise ValueError(f"f {tuple(f.shape)} must have x's shape {tuple(shape)}")
        grad = grad or f.requires_grad
    if (post_bias is not None and post_weight is None) or (pre_bias is not None and pre_weight is None):
        raise ValueError("a norm's bias needs its weight")
    params, params_dtype = [post_weight, post_bias, scale, pre_weight, pre_bias], None
    for i, t in enumerate(params):
        if t is not None:
            name = _PARAMS[i]
            check(t, name, mixed if params_dtype is None else _native.ALONE[params_dtype], gpu)
            params_dtype = t.dtype
            if t.dim() != 1 or t.shape[0] != width:
                raise ValueError(f"{name} must have shape ({width},), got {tuple(t.shape)}")
            params[i] = t.contiguous()
            grad = grad or t.requires_grad
    # the common case, matrices, adds no view to the graph
    flat = len(shape) == 2
    mode = 0
    if gate is not None:
        check(gate, "gate", mixed, gpu)
        gate_shape, lead = gate.shape, shape[:-1]
        if gate_shape == lead or (gate_shape == lead + (1,) and width > 1):
            mode = 1
            if len(gate_shape) == len(lead) and gate.numel() > 1 and \
                    all(n in (1, to) for n, to in zip(gate_shape, shape[1:])):
                raise ValueError(f"gate {tuple(gate_shape)} could be per row or per column of x {tuple(shape)}: give it "
                                 f"as {tuple(gate_shape) + (1,)} or as {(1,) + tuple(gate_shape)}")
            if gate.dim() != 1:
                gate = gate.reshape(-1)
        else:
            mode = 2
            check(gate, "gate", alone, gpu)
            if gate.shape != shape:
                try:
                    gate = gate.expand(shape)
                except RuntimeError:
                    raise ValueError(f"gate {tuple(gate.shape)} fits neither x's rows nor its shape {tuple(shape)}") \
                        from None
            if not flat:
                gate = gate.reshape(-1, width)
        gate = gate.contiguous()
        grad = grad or gate.requires_grad
    x2 = (x if flat else x.reshape(-1, width)).contiguous()
    f2 = None if f is None else (f if flat else f.reshape(-1, width)).contiguous()
    meta = (_KINDS[kind], mode, gate_activation == "sigmoid", scale_value, float(eps),
            _native.DTYPES[params_dtype or dt], _native.DTYPES[dt if gate is None else gate.dtype])
    if _native.differentiates(grad):
        y, h = BlockNormFunction.apply(x2, f2, gate, *params, meta)
    else:
        y, h, _ = _forward(x2, f2, gate, params, meta, False)
    if f is None:
        y = x
    elif not flat:
        y = y.view(shape)
    return y, h if h is None or flat else h.view(shape)
