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
