"""The block-FP8 and layer norm entry points without a GPU: what they refuse,
and the workspaces they ask for (include/nflow_block.h)."""
import ctypes as C

import pytest
import torch

from neuroflow_amd import _lib
from neuroflow_amd import block_fp8 as B
from neuroflow_amd import norm as L

P = 4096           # a non-null, aligned address; never followed: every call here is refused or has no work


def call(name, *args):
    return getattr(_lib.lib(), name)(*args)


def ok_and_refused(name, good, bad):
    """`good` (with no rows, so no work) passes; every replacement in `bad` is
    refused with a message that names the entry point."""
    assert call(name, *good) == _lib.OK
    for at, value in bad:
        args = list(good)
        for i, v in zip(at if isinstance(at, tuple) else (at,), value if isinstance(at, tuple) else (value,)):
            args[i] = v
        assert call(name, *args) == _lib.INVALID_ARG, (name, at, value)
        assert name[len("nflow_"):].encode() in _lib.lib().nflow_last_error(), name


def test_layer_norm_forward():
    #       x  dtype M  D   ldx w     b     eps   y  ldy mean  rstd  stream
    good = [P, 0, 0, 64, 64, None, None, 1e-5, P, 64, None, None, None]
    ok_and_refused("nflow_layer_norm_forward", good,
                   [(1, 2), (1, -1), (2, -1), (3, 0), (4, 63), (7, -1.0), (7, float("nan")), (9, 63), ((2, 0), (1, None)),
                    ((2, 8), (1, None))])


def test_layer_norm_fp8_block():
    good = [P, 1, 0, 64, 64, None, None, 1e-5, P, P, None, None, None]
    ok_and_refused("nflow_layer_norm_fp8_block", good,
                   [(1, 5), (3, 0), (4, 10), (7, -0.5), ((2, 8), (1, None)), ((2, 9), (1, None)), ((2, 8), (1, P + 8))])


def test_layer_norm_backward():
    #       dy x  dtype M D lddy ldx w mean rstd dx lddx dw db ws n stream
    good = [P, P, 0, 0, 64, 64, 64, None, P, P, P, 64, None, None, None, 0, None]
    n = C.c_size_t()
    assert call("nflow_layer_norm_backward_workspace", 10, 64, C.byref(n)) == _lib.OK and n.value >= 2 * 64 * 4
    need = n.value
    ok_and_refused("nflow_layer_norm_backward", good,
                   [(2, 9), (3, -1), (4, 0), (5, 63), (6, 63), (11, 63), ((3, 0, 14, 15), (10, None, P, need)),
                    ((3, 8, 14, 15), (10, None, P, need)), ((3, 10, 14, 15), (10, None, P, need)),
                    ((3, 14, 15), (10, None, 0)), ((3, 14, 15), (10, P, need - 1)), ((3, 14, 15), (10, P + 4, need))])
    assert call("nflow_layer_norm_backward_workspace", 10, 0, C.byref(n)) == _lib.INVALID_ARG
    assert call("nflow_layer_norm_backward_workspace", 10, 64, None) == _lib.INVALID_ARG


def test_quantise():
    good = [P, 0, 0, 64, 64, P, P, None, None, None]
    ok_and_refused("nflow_fp8_block_quantise", good,
                   [(1, 3), (2, -1), (3, -1), (4, 63), ((2, 0), (1, None)), ((2, 5, 6), (1, None, None)),
                    ((2, 6), (1, None)), ((2, 7), (1, P)), ((2, 5), (1, P + 1))])
    good = [P, 0, 0, 64, 64, P, P, None, None, None]
    ok_and_refused("nflow_fp8_block_quantise_weight", good,
                   [(1, 3), (2, -1), (4, 63), ((2, 0), (1, None)), ((2, 5), (1, None)), ((2, 8), (1, P))])


def test_products():
    #       A  sA W  sW blk M N  K    bias act C dtype ldc ws n stream
    good = [P, P, P, P, 1, 0, 8, 256, None, 0, P, 0, 8, None, 0, None]
    ok_and_refused("nflow_fp8_block_matmul", good,
                   [(5, -1), (6, -1), (7, -1), (7, (1 << 22) + 1), (9, 3), (9, -1), (11, 2), (12, 7), ((5, 0), (1, None)),
                    ((5, 1), (1, None)), ((5, 2), (1, None)), ((5, 3), (1, None)), ((5, 10), (1, None)), ((5, 0), (1, P + 8)),
                    ((5, 6, 12), (1 << 40, 1 << 20, 1 << 20))])
    #       x dtype M K ldx W sW N bias act y ldy ws n stream
    good = [P, 0, 0, 256, 256, P, P, 8, None, 0, P, 8, None, 0, None]
    ok_and_refused("nflow_fp8_block_linear", good,
                   [(1, 2), (2, -1), (4, 255), (9, 7), (11, 7), ((2, 0), (1, None)), ((2, 5), (1, None)), ((2, 10), (1, None)),
                    (2, 1000)])          # 1000 rows need a workspace
    #       dy dtype M N lddy x_t s W_t s K dx lddx dW db ws n stream
    good = [P, 0, 0, 8, 8, P, P, P, P, 256, None, 256, None, None, P, 1 << 30, None]
    ok_and_refused("nflow_fp8_block_linear_backward", good,
                   [(1, 2), (2, -1), (4, 7), ((2, 0), (1, None)), ((2, 10, 11), (1, P, 255)), ((2, 10, 7), (1, P, None)),
                    ((2, 12, 5), (1, P, None)), ((2, 10, 14, 15), (1, P, None, 0))])


def test_workspace_queries():
    n = C.c_size_t(1)
    for name in ("matmul", "linear", "linear_backward"):
        f = f"nflow_fp8_block_{name}_workspace"
        assert call(f, 1000, 512, 384, 0, C.byref(n)) == _lib.OK
        assert call(f, 1000, 512, 384, 0, None) == _lib.INVALID_ARG
        assert call(f, -1, 512, 384, 0, C.byref(n)) == _lib.INVALID_ARG and n.value == 0
        assert call(f, 1000, 512, 384, 7, C.byref(n)) == _lib.INVALID_ARG
        assert call(f, 0, 0, 0, 1, C.byref(n)) == _lib.OK and n.value == 0
    # One row is quantised where it is multiplied; many rows' codes need room.
    assert call("nflow_fp8_block_linear_workspace", 1, 4096, 4096, 1, C.byref(n)) == _lib.OK and n.value == 0
    assert call("nflow_fp8_block_linear_workspace", 5000, 256, 256, 1, C.byref(n)) == _lib.OK and n.value >= 5000 * 256


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 256)
    for f in (lambda: B.quantise(x), lambda: B.quantise_both(x), lambda: B.quantise_weight(x), lambda: L.layer_norm(x),
              lambda: L.layer_norm_fp8(x), lambda: L.layer_norm_backward(x, x, None, x[:, 0], x[:, 0])):
        with pytest.raises(TypeError):
            f()
    q = B.BlockFp8(torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(2, 4), 256)
    with pytest.raises(TypeError):
        B.matmul(q, q)
