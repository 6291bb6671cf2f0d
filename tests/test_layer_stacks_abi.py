"""libnnue_ls.so loads, exports what include/nnue_ls.h declares, its structs
match the binding's, and bad arguments are refused on the host."""

import ctypes
import os
import re

import pytest
import torch

from stockfish_trainer_b200 import layer_stacks
from stockfish_trainer_b200.layer_stacks import _native

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "nnue_ls.h")


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_library_exports_every_declared_symbol():
    names = sorted(set(re.findall(r"\b(nnue_ls_\w+)\s*\(", _text())))
    assert len(names) >= 12 and names == sorted(_native.exported_symbols())
    lib = _native.load()
    for name in names:
        assert hasattr(lib, name), name
    assert lib.nnue_ls_version() >= 100


@pytest.mark.parametrize("struct,name", [(_native.Linear, "nnue_ls_linear"), (_native.Norm, "nnue_ls_norm"),
                                         (_native.Route, "nnue_ls_route")])
def test_struct_fields_match_the_header(struct, name):
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", _text()).group(1)
    widths = {"int64_t": 8, "int32_t": 4, "float": 4}
    fields = []
    for decl in body.split(";"):
        decl = decl.replace("const ", "").strip()
        if decl:
            kind, rest = decl.split(None, 1)
            for var in rest.split(","):
                var = var.strip()
                fields.append((var.lstrip("*").strip(), 8 if "*" in var else widths[kind]))
    assert fields == [(n, ctypes.sizeof(t)) for n, t in struct._fields_]


def _linear(**kw):
    a = _native.Linear(rows=4, inputs=8, outputs=8, ldx=8, ldw=8, ldr=8, ldg=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_linear_refusals():
    lib = _native.load()
    some = 4096  # never dereferenced

    def fwd(a):
        return lib.nnue_ls_linear_forward(ctypes.byref(a), None, 0, None)

    assert lib.nnue_ls_linear_forward(None, None, 0, None) == _native.ERR_INVALID_ARGUMENT
    assert fwd(_linear()) == _native.ERR_INVALID_ARGUMENT and "null" in _native.last_error()
    good = dict(x=some, weight=some, out=some)
    for bad in (dict(rows=-1), dict(inputs=0), dict(outputs=0), dict(dtype=3), dict(bias_dtype=2), dict(activation=6),
                dict(activation=-1), dict(ldx=7), dict(ldw=7), dict(residual=some, ldr=7)):
        assert fwd(_linear(**good, **bad)) == _native.ERR_INVALID_ARGUMENT, bad
    assert fwd(_linear(rows=2**30, **good)) == _native.ERR_UNSUPPORTED
    assert fwd(_linear(rows=0)) == _native.OK
    a = _linear(x=some, weight=some, grad_out=some, grad_x=some, activation=4)
    assert lib.nnue_ls_linear_backward(ctypes.byref(a), None, 0, None) == _native.ERR_INVALID_ARGUMENT  # no act_grad
    a.act_grad = some
    need = lib.nnue_ls_linear_backward_workspace_size(ctypes.byref(a))
    assert need > 0
    assert lib.nnue_ls_linear_backward(ctypes.byref(a), some, need - 1, None) == _native.ERR_WORKSPACE
    assert lib.nnue_ls_linear_backward(ctypes.byref(a), some + 8, need, None) == _native.ERR_WORKSPACE


def test_linear_saved_layout():
    """act'(z), x and the weight in one buffer: only what is asked for and needed, 256-byte aligned, no overlap."""
    lib = _native.load()
    off = (ctypes.c_int64 * 3)()
    a = _linear(rows=100, inputs=40, outputs=24, ldx=40, ldw=40, x=4096, weight=4096, activation=4)
    total = lib.nnue_ls_linear_saved_layout(ctypes.byref(a), 7, off)  # fp32: all three
    assert list(off) == [0, 9728, 9728 + 24064] and total == 9728 + 24064 + 5888
    assert lib.nnue_ls_linear_saved_layout(ctypes.byref(a), 2, off) == 24064 and list(off) == [-1, 0, -1]
    a.dtype = a.bias_dtype = 1  # aligned 16-bit operands are read as they lie
    assert lib.nnue_ls_linear_saved_layout(ctypes.byref(a), 7, off) == 4864 and list(off) == [0, -1, -1]
    a.ldx = 41
    assert lib.nnue_ls_linear_saved_layout(ctypes.byref(a), 6, off) == 8192 and list(off) == [-1, 0, -1]
    a.activation = 0
    assert lib.nnue_ls_linear_saved_layout(ctypes.byref(a), 1, off) == 0
    a.x_packed = 4096 + 8
    a.out = 4096
    assert lib.nnue_ls_linear_forward(ctypes.byref(a), None, 0, None) == _native.ERR_INVALID_ARGUMENT
    a.x_packed, a.ldx = 4096, 40  # a buffer for an x that is not packed
    assert lib.nnue_ls_linear_forward(ctypes.byref(a), None, 0, None) == _native.ERR_INVALID_ARGUMENT


def test_norm_refusals():
    lib = _native.load()
    some = 4096

    def fwd(**kw):
        a = _native.Norm(**{**dict(rows=4, width=8, x=some, f=some, y=some, post_weight=some, eps=1e-5), **kw})
        return lib.nnue_ls_norm_forward(ctypes.byref(a), None)

    for bad in (dict(rows=-1), dict(width=0), dict(dtype=3), dict(kind=2), dict(gate_mode=3), dict(gate_mode=1),
                dict(f=None), dict(x=None), dict(y=None), dict(pre_bias=some), dict(pre_weight=some), dict(h=some),
                dict(post_weight=None, post_bias=some), dict(eps=-1.0), dict(eps=float("nan")), dict(params_dtype=1)):
        assert fwd(**bad) == _native.ERR_INVALID_ARGUMENT, bad
    assert fwd(width=_native.NORM_MAX_WIDTH + 1) == _native.ERR_UNSUPPORTED
    assert fwd(rows=0) == _native.OK
    a = _native.Norm(rows=4, width=8, x=some, f=some, stats=some, eps=1e-5, post_weight=some, grad_post_weight=some)
    need = lib.nnue_ls_norm_backward_workspace_size(ctypes.byref(a))
    assert need > 0
    assert lib.nnue_ls_norm_backward(ctypes.byref(a), some, need - 1, None) == _native.ERR_WORKSPACE


def test_route_refusals():
    lib = _native.load()
    some = 4096

    def fwd(ws=some, size=1 << 20, **kw):
        a = _native.Route(**{**dict(rows=4, experts=8, k=2, ld=8, logits=some, indices=some, gates=some, counts=some,
                                    loss=some), **kw})
        return lib.nnue_ls_route_forward(ctypes.byref(a), ws, size, None)

    for bad in (dict(rows=-1), dict(experts=0), dict(k=0), dict(k=9), dict(dtype=3), dict(logits=None), dict(ld=7),
                dict(indices=None), dict(gates=None), dict(counts=None), dict(loss=None)):
        assert fwd(**bad) == _native.ERR_INVALID_ARGUMENT, bad
    assert fwd(experts=_native.MAX_EXPERTS + 1, ld=2048) == _native.ERR_UNSUPPORTED
    assert fwd(size=0) == _native.ERR_WORKSPACE and fwd(ws=None) == _native.ERR_WORKSPACE


def test_python_refusals_without_a_gpu():
    """The wrappers check type and place before they look at anything else."""
    x = torch.zeros(2, 8)
    for call in (lambda: layer_stacks.linear_act(x, x), lambda: layer_stacks.block_norm(x, pre_weight=x[0]),
                 lambda: layer_stacks.route(x, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: layer_stacks.linear_act(x.double(), x.double()), lambda: layer_stacks.route(x.long(), 1),
                 lambda: layer_stacks.block_norm([1.0])):
        with pytest.raises(TypeError):
            call()
