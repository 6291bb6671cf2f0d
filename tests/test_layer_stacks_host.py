"""Host side of libnnue_ls.so at the limits of its arguments (no GPU needed)."""

import ctypes

import pytest

from stockfish_trainer_b200.layer_stacks import _native

SOME = 4096  # an address that is never dereferenced


@pytest.mark.parametrize("dtype", range(3))
@pytest.mark.parametrize("wanted", [("grad_x",), ("grad_weight",), ("grad_bias",), ("grad_x", "grad_weight", "grad_bias")])
def test_linear_backward_of_no_rows_plans_nothing(dtype, wanted):
    a = _native.Linear(rows=0, inputs=16, outputs=8, ldx=16, ldw=16, ldg=8, dtype=dtype, bias_dtype=dtype, activation=4,
                       x=SOME, weight=SOME, grad_out=SOME, act_grad=SOME, **{name: SOME for name in wanted})
    assert _native.load().nnue_ls_linear_backward_workspace_size(ctypes.byref(a)) == 0


def _refused(func, args, *rest):
    rc = getattr(_native.load(), func)(ctypes.byref(args), *rest)
    return rc == _native.ERR_INVALID_ARGUMENT and "aligned" in _native.last_error()


_MATRICES = ("x", "weight", "residual", "out", "act_grad", "grad_out", "grad_x", "grad_weight")


@pytest.mark.parametrize("dtype,bias_dtype", [(0, 0), (1, 1), (2, 0)])
def test_misaligned_pointers_of_a_linear_call(dtype, bias_dtype):
    """Refused on the host: on the device they would fault."""
    for name in (*_MATRICES, "bias", "grad_bias"):
        size = 4 if (bias_dtype if "bias" in name else dtype) == 0 else 2
        good = dict(rows=100, inputs=16, outputs=8, ldx=16, ldw=16, ldr=8, ldg=8, dtype=dtype, bias_dtype=bias_dtype,
                    activation=4, **{n: SOME for n in _MATRICES})
        for step in range(1, size):
            a = _native.Linear(**{**good, name: SOME + step})
            assert _refused("nnue_ls_linear_forward", a, None, 0, None), (name, step)
            assert _refused("nnue_ls_linear_backward", a, None, 0, None), (name, step)
    for name in ("x_packed", "weight_packed"):
        a = _native.Linear(**{**good, name: SOME + 128})
        assert _refused("nnue_ls_linear_forward", a, None, 0, None)
        assert _refused("nnue_ls_linear_backward", a, None, 0, None)


_ROWS = ("x", "f", "y", "h", "grad_y", "grad_h", "grad_x", "grad_f")
_PARAMS = ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias", "grad_post_weight", "grad_post_bias",
           "grad_scale", "grad_pre_weight", "grad_pre_bias")


@pytest.mark.parametrize("dtype,params_dtype,gate_dtype,gate_mode", [(0, 0, 0, 2), (1, 1, 1, 1), (2, 0, 0, 1), (1, 0, 0, 2)])
def test_misaligned_pointers_of_a_norm_call(dtype, params_dtype, gate_dtype, gate_mode):
    good = dict(rows=3, width=8, dtype=dtype, params_dtype=params_dtype, gate_dtype=gate_dtype, gate_mode=gate_mode,
                eps=1e-5, stats=SOME, gate=SOME, grad_gate=SOME, **{n: SOME for n in _ROWS + _PARAMS})
    for name in (*_ROWS, *_PARAMS, "gate", "grad_gate", "stats"):
        code = params_dtype if name in _PARAMS else gate_dtype if "gate" in name and gate_mode == 1 else dtype
        size = 16 if name == "stats" else 4 if code == 0 else 2
        for step in range(1, size):
            a = _native.Norm(**{**good, name: SOME + step})
            assert _refused("nnue_ls_norm_forward", a, None), (name, step)
            assert _refused("nnue_ls_norm_backward", a, None, 0, None), (name, step)


@pytest.mark.parametrize("dtype", range(3))
def test_misaligned_pointers_of_a_route_call(dtype):
    sizes = {"logits": 2 if dtype else 4, "grad_logits": 2 if dtype else 4, "indices": 8, "counts": 8, "gates": 4, "loss": 4,
             "grad_gates": 4, "grad_loss": 4}
    for name, size in sizes.items():
        for step in range(1, size):
            a = _native.Route(rows=4, experts=8, k=2, ld=8, dtype=dtype, **{**dict.fromkeys(sizes, SOME), name: SOME + step})
            assert _refused("nnue_ls_route_forward", a, None, 0, None), (name, step)
            assert _refused("nnue_ls_route_backward", a, None), (name, step)
