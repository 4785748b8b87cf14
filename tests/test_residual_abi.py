"""The entry points of include/nflow_residual.h without a GPU: what they refuse,
and the workspaces they ask for."""
import ctypes as C

import pytest
import torch

from neuroflow_amd import _lib, dense, grads
from neuroflow_amd import norm as L

P = 1 << 20        # a non-null, aligned address; never followed: every call here is refused or has no work
Q, R, S = 2 * P, 3 * P, 4 * P


def call(name, *args):
    return getattr(_lib.lib(), name)(*args)


def ok_and_refused(name, good, bad):
    """`good` (with no rows, so no work) passes; every replacement in `bad` is
    refused with a message that names the entry point."""
    assert call(name, *good) == _lib.OK, _lib.lib().nflow_last_error()
    for at, value in bad:
        args = list(good)
        for i, v in zip(at if isinstance(at, tuple) else (at,), value if isinstance(at, tuple) else (value,)):
            args[i] = v
        assert call(name, *args) == _lib.INVALID_ARG, (name, at, value)
        assert name[len("nflow_"):].encode() in _lib.lib().nflow_last_error(), name


def test_every_entry_point_is_bound():
    from neuroflow_amd import block_fp8
    names = set(block_fp8._ops().residual_entry_points())
    assert names == {n for n in _lib.SIGNATURES if n.startswith(("nflow_rms_", "nflow_dense_", "nflow_grad_"))}


def test_rms_norm_forward():
    #       x dtype M D ldx r   ldr w     eps  y  ldy sum   lds rstd  stream
    good = [P, 0, 0, 64, 64, Q, 64, None, 1e-5, R, 64, S, 64, None, None]
    ok_and_refused("nflow_rms_norm_forward", good,
                   [(1, 2), (2, -1), (3, 0), (4, 63), (6, 63), (8, -1.0), (8, float("nan")), (10, 63), (12, 63), (5, None),
                    ((2, 0), (1, None)), ((2, 9), (1, None)), ((2, 9), (2, S)), ((2, 9), (2, S + 256)), ((2, 11), (8, P + 256)),
                    ((2, 11), (8, Q - 256)), ((2, 9), (8, P + 4)), ((2, 9, 10), (8, P, 65)), ((2, 9, 10), (8, Q, 72))])


def test_rms_norm_fp8():
    good = [P, 1, 0, 64, 64, Q, 64, None, 1e-5, R, R, S, 64, None, None]
    ok_and_refused("nflow_rms_norm_fp8", good,
                   [(1, 5), (3, -4), (4, 10), (8, -0.5), ((2, 9), (1, None)), ((2, 10), (1, None)), ((2, 9), (1, R + 8)),
                    ((2, 11), (8, Q + 64)), (5, None)])


def test_rms_norm_backward():
    n = C.c_size_t()
    assert call("nflow_rms_norm_backward_workspace", 10, 64, C.byref(n)) == _lib.OK and n.value >= 64 * 4
    need = n.value
    #       dy t dtype M D lddy ldt w     rstd ds ldds dt lddt dw    ws    n  stream
    good = [P, Q, 0, 0, 64, 64, 64, None, S, None, 64, R, 64, None, None, 0, None]
    full = (10, None, P, need)
    ok_and_refused("nflow_rms_norm_backward", good,
                   [(2, 9), (3, -1), (4, 0), (5, 63), (6, 63), (12, 63), ((9, 10), (S, 63)), ((3, 0, 14, 15), full),
                    ((3, 8, 14, 15), full), ((3, 11, 14, 15), full), ((3, 14, 15), (10, None, 0)), ((3, 14, 15), (10, S, need - 1)),
                    ((3, 14, 15), (10, S + 4, need)), ((3, 11, 14, 15), (10, P + 256, S, need)),
                    ((3, 9, 11, 14, 15), (10, R + 128, R, S, need))])
    assert call("nflow_rms_norm_backward_workspace", 10, 0, C.byref(n)) == _lib.INVALID_ARG
    assert call("nflow_rms_norm_backward_workspace", 10, 64, None) == _lib.INVALID_ARG


def test_dense_linear():
    #       x dtype M K ldx W ldw N bias  r     ldr act y ldy pre   ldp ws    n  stream
    good = [P, 0, 0, 64, 64, Q, 64, 8, None, None, 8, 0, R, 8, None, 8, None, 0, None]
    ok_and_refused("nflow_dense_linear", good,
                   [(1, 2), (2, -1), (3, -1), (7, -1), (4, 63), (6, 63), (11, 3), (11, -1), (13, 7), ((9, 10), (S, 7)),
                    ((14, 15), (S, 7)), ((2, 0), (4, None)), ((2, 5), (4, None)), ((2, 12), (4, None)), ((2, 12), (4, P)),
                    ((2, 12), (4, Q + 16)), ((2, 14), (4, R)), ((2, 14), (4, P)), ((2, 9), (4, R + 32)),
                    ((2, 9, 14), (4, S, S)), ((2, 9, 10), (4, R, 16)), (3, (1 << 21) + 1), ((2, 7, 13), (1 << 40, 1 << 20, 1 << 20))])
    # A tile's operands off 16-byte alignment need the room for their copies.
    n = C.c_size_t()
    assert call("nflow_dense_linear_workspace", 100, 8, 64, 1, 0, C.byref(n)) == _lib.OK
    plain = n.value
    assert call("nflow_dense_linear_workspace", 100, 8, 64, 1, 1, C.byref(n)) == _lib.OK and n.value >= plain + 2 * 108 * 64
    args = [P + 2, 1, 100, 64, 64, Q, 64, 8, None, None, 8, 0, R, 8, None, 8, S if plain else None, plain, None]
    assert call("nflow_dense_linear", *args) == _lib.INVALID_ARG


def test_dense_linear_backward():
    #       dy dtype M N lddy x ldx W ldw K act pre  ldp dz    lddz dx lddx dW lddw db    ws    n  stream
    good = [P, 0, 0, 8, 8, Q, 64, R, 64, 64, 0, None, 8, None, 8, None, 64, None, 64, None, None, 0, None]
    ok_and_refused("nflow_dense_linear_backward", good,
                   [(1, 2), (2, -1), (3, -1), (9, -1), (4, 7), (10, 9), (11, S), (13, S), ((15, 16), (S, 63)), ((15, 8), (S, 63)),
                    ((17, 18), (S, 63)), ((17, 6), (S, 63))])
    n = C.c_size_t()
    for copies in (0, 1):
        assert call("nflow_dense_linear_backward_workspace", 16, 8, 64, 0, copies, C.byref(n)) == _lib.OK
    ws, need = 64 * P, n.value
    good[2], good[20], good[21] = 16, ws, need
    bad = [((0, 15), (None, S)), ((15, 7), (S, None)), ((17, 5), (S, None)), ((10, 11, 13), (1, None, S)),
           ((10, 11, 13), (1, S, None)), ((15, 20, 21), (S, None, 0)), ((15, 21), (S, need - 1)), (15, P), ((15, 17), (S, S + 64)),
           (17, Q), ((10, 11, 13), (1, S, S + 16)), ((10, 11, 13, 14), (1, S, S, 9)), ((10, 11, 13, 17), (1, S, Q, S + P)),
           ((10, 11, 13, 15), (1, S, 5 * P, 5 * P))]
    for at, value in bad:
        args = list(good)
        for i, v in zip(at if isinstance(at, tuple) else (at,), value if isinstance(at, tuple) else (value,)):
            args[i] = v
        assert call("nflow_dense_linear_backward", *args) == _lib.INVALID_ARG, (at, value)


def test_dense_workspace_queries():
    n = C.c_size_t(1)
    for name in ("linear", "linear_backward"):
        f = f"nflow_dense_{name}_workspace"
        assert call(f, 1000, 512, 384, 0, 0, C.byref(n)) == _lib.OK
        assert call(f, 1000, 512, 384, 0, 0, None) == _lib.INVALID_ARG
        assert call(f, -1, 512, 384, 0, 0, C.byref(n)) == _lib.INVALID_ARG and n.value == 0
        assert call(f, 1000, 512, 384, 7, 0, C.byref(n)) == _lib.INVALID_ARG
        assert call(f, 0, 0, 0, 1, 0, C.byref(n)) == _lib.OK and n.value == 0
    assert call("nflow_dense_linear_workspace", 1, 4096, 4096, 1, 1, C.byref(n)) == _lib.OK and n.value == 0   # few rows: none


def table(*tensors):
    return (_lib.GradTensorC * len(tensors))(*(_lib.GradTensorC(g, o, c, d) for g, o, c, d in tensors))


def test_grads():
    n = C.c_size_t()
    assert call("nflow_grad_workspace", 3, C.byref(n)) == _lib.OK and n.value > 0
    ws, need = 64 * P, n.value
    assert call("nflow_grad_workspace", -1, C.byref(n)) == _lib.INVALID_ARG
    assert call("nflow_grad_workspace", 3, None) == _lib.INVALID_ARG
    one = (P, P, 100, 0)
    def refused(t, count=None, norm=Q, max_norm=1.0, w=ws, size=need, both=True):
        count = len(t) if count is None else count
        if both:
            assert call("nflow_grad_norm", t, count, norm, w, size, None) == _lib.INVALID_ARG
            assert b"grad_norm" in _lib.lib().nflow_last_error()
        assert call("nflow_grad_clip", t, count, max_norm, norm, w, size, None) == _lib.INVALID_ARG
        assert b"grad_clip" in _lib.lib().nflow_last_error()
    refused(table(one), norm=None)
    refused(table(one), count=-1)
    refused(None, count=1)
    refused(table((P, P, 100, 2)))
    refused(table((P, P, -1, 0)))
    refused(table((None, P, 1, 0)))
    refused(table((P, P, 1 << 50, 0)))
    refused(table(one), w=None)
    refused(table(one), w=ws + 8)
    refused(table(one), size=need - 1)
    refused(table(one), max_norm=-1.0, both=False)
    refused(table(one), max_norm=float("nan"), both=False)
    refused(table((P, None, 1, 0)), both=False)
    for other in ((P, P, 1, 0), (P + 396, P + 396, 1, 0), (R, P + 396, 1, 0), (P + 396, R, 1, 0), (R, R + 4, 2, 0), (P - 2, P - 2, 2, 1)):
        refused(table(one, other), both=False)
    # None of these: side by side, and the memory of one tensor's grad to another place.
    assert call("nflow_grad_clip", table((P, P, 0, 0), (P, P, 0, 0)), 2, 1.0, None, ws, need, None) == _lib.INVALID_ARG


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 64)
    for f in (lambda: L.rms_norm(x), lambda: L.rms_norm_fp8(x), lambda: L.rms_norm_backward(x, x, None, x[:, 0]),
              lambda: dense.linear(x, x), lambda: dense.linear_backward(x, x, x), lambda: grads.global_norm([x]),
              lambda: grads.clip_by_global_norm([x], 1.0)):
        with pytest.raises(TypeError):
            f()
    with pytest.raises(ValueError):
        grads.global_norm([])
