"""Results that share memory with a vector of the call, or with another result, are
refused ahead of any launch: no GPU is needed for that, and no address of those tests is followed."""
import ctypes as C

import pytest
import torch

from neuroflow_amd import _lib, norm

P = 1 << 24
M, D, N, K = 6, 256, 40, 64
X, R, Y, S, W, RS, CODES, SCALES, WS = (P * (i + 1) for i in range(9))


def refused(name, args, what=b"shares memory"):
    assert getattr(_lib.lib(), name)(*args) == _lib.INVALID_ARG
    assert what in _lib.lib().nflow_last_error(), _lib.lib().nflow_last_error()


# What is moved, and to where: on a vector, on its last value, and a row of it that ends on it.
@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2)])
@pytest.mark.parametrize("y,s,w,rs", [(W, S, W, RS), (Y, W, W, RS), (Y, S, Y + 4 * (D - 1), RS), (Y, S, S + 4 * (D - 1), RS),
                                      (Y, S, W, X), (Y, S, W, R + 8), (Y, S, W, Y + 64), (Y, S, W, S + 64), (Y, S, W, W + 4 * (D - 1)),
                                      (Y, S, S - 4 * (D - 1), RS)])
def test_rms_norm(dtype, size, y, s, w, rs):
    refused("nflow_rms_norm_forward", [X, dtype, M, D, D, R, D, w, 1e-5, y, D, s, D, rs, None])


@pytest.mark.parametrize("codes,scales,s,w,rs", [
    (X, SCALES, S, W, RS), (R, SCALES, S, W, RS), (CODES, R + 16, S, W, RS), (CODES, X + 16, S, W, RS), (CODES, SCALES, W, W, RS),
    (S, SCALES, S, W, RS), (CODES, S + 16, S, W, RS), (W, SCALES, S, W, RS), (CODES, W + 4 * (D - 1), S, W, RS),
    (CODES, CODES + M * D - 4, S, W, RS), (CODES, SCALES, S, W, CODES), (CODES, SCALES, S, W, SCALES + 4 * (2 * M - 1)),
    (CODES, SCALES, S, W, W), (CODES, SCALES, S, W, X)])
def test_rms_norm_fp8(codes, scales, s, w, rs):
    refused("nflow_rms_norm_fp8", [X, 1, M, D, D, R, D, w, 1e-5, codes, scales, s, D, rs, None])


def test_rms_norm_backward():
    n = C.c_size_t()
    assert _lib.lib().nflow_rms_norm_backward_workspace(M, D, C.byref(n)) == _lib.OK
    DY, T, DS, DT, DW = X, R, S, Y, CODES
    for dt, dw, w in ((W, DW, W), (RS, DW, W), (DT, DT, W), (DT, DY, W), (DT, T + 8, W), (DT, DS, W), (DT, W, W), (DT, RS, W),
                      (DT, DT + 4 * (M * D - 1), W), (DT, DT - 4 * (D - 1), W)):
        refused("nflow_rms_norm_backward", [DY, T, 0, M, D, D, D, w, RS, DS, D, dt, D, dw, WS, n.value, None])


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("y,pre", [(W, S), (Y, W), (W + 4 * (N - 1), S), (Y, W - 8), (W - 2 * (M * N - 2), S)])
def test_dense_linear(dtype, y, pre):
    """The results and the bias."""
    n = C.c_size_t()
    assert _lib.lib().nflow_dense_linear_workspace(M, N, K, dtype, 1, C.byref(n)) == _lib.OK
    refused("nflow_dense_linear", [X, dtype, M, K, K, R, K, N, W, None, 0, 2, y, N, pre, N, WS, n.value, None])


def test_dense_linear_backward():
    """dbias and everything else."""
    n = C.c_size_t()
    assert _lib.lib().nflow_dense_linear_backward_workspace(M, N, K, 0, 1, C.byref(n)) == _lib.OK
    DY, PRE, DZ, DX, DW = S, RS, Y, CODES, SCALES
    for db in (DY, X, R, PRE, DZ, DX, DW, DX + 4 * (M * K - 1), DW - 4 * (N - 1), X + 4 * K):
        refused("nflow_dense_linear_backward", [DY, 0, M, N, N, X, K, R, K, K, 2, PRE, N, DZ, N, DX, K, DW, K, db, WS, n.value, None])


@pytest.mark.parametrize("norm", [X, X + 396, X - 2, Y, Y + 396, S + 2])
def test_grad_clip(norm):
    """The norm and a gradient in place, another's out, and a bf16 one."""
    n = C.c_size_t()
    assert _lib.lib().nflow_grad_workspace(3, C.byref(n)) == _lib.OK
    t = (_lib.GradTensorC * 3)(*(_lib.GradTensorC(*v) for v in ((X, X, 100, 0), (R, Y, 100, 0), (S, S, 2, 1))))
    refused("nflow_grad_clip", [t, 3, 1.0, norm, WS, n.value, None], b"overlaps")


def test_vectors_on_rows():
    """A vector in the gap between rows, one value too far in either direction."""
    ld = 3 * D
    for at in (Y + 4 * (D - 1), Y + 4 * (2 * D + 1), Y - 4 * (D - 1), Y + 4 * (ld * (M - 1) + D - 1)):
        refused("nflow_rms_norm_forward", [X, 0, M, D, D, None, 0, at, 1e-5, Y, ld, None, 0, None, None])


@pytest.mark.gpu
def test_vectors_between_rows(gpu):
    """There, and on either side of all rows, it shares no memory with them."""
    g = torch.Generator(device="cuda").manual_seed(1)
    buf = torch.full((M, 3 * D), 7.0, device="cuda")
    r = torch.randn(M, D, generator=g, device="cuda")
    x, to = torch.randn(M, D, generator=g, device="cuda"), buf[:, D:2 * D]
    want = None
    for w in (buf[0, :D], buf[0, 2 * D:], buf[3, 2 * D:], buf.view(-1)[5 * D:6 * D], buf[M - 1, 2 * D:]):
        w.copy_(torch.linspace(0.5, 2, D, device="cuda"))
        y, t = norm.rms_norm(x, w, residual=r, sum_out=to)
        want = y.clone() if want is None else want
        assert torch.equal(y, want) and torch.equal(t, x + r)
