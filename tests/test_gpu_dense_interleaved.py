"""Operands and results that are columns of one buffer share rows' strides but no
memory: taken like any others, and what lies between them is left as it was."""
import ctypes as C

import pytest
import torch

from neuroflow_amd import _lib, dense
from residual_reference import DTYPES, act, act_bound, dense_bound, gen, half, rows, within
from residual_reference import dense as product

pytestmark = pytest.mark.gpu
SIZES = [(1, 40, 24), (20, 64, 40), (33, 100, 72), (300, 513, 260), (700, 256, 512)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("gap", [0, 3, 8])
def test_forward(gpu, M, K, N, dtype, gap):
    g = gen(M + gap)
    buf = torch.full((M, K + 2 * N + 3 * gap + (gap != 8)), 7.0, device="cuda", dtype=dtype)
    x, r, y = buf[:, :K], buf[:, K + gap:K + gap + N], buf[:, K + 2 * gap + N:K + 2 * gap + 2 * N]
    x.copy_(rows(M, K, dtype, g))
    r.copy_(rows(M, N, dtype, g, 0.5))
    W, b = rows(N, K, dtype, g, K ** -0.5), torch.randn(N, generator=g, device="cuda")
    before = buf.clone()
    assert dense.linear(x, W, b, "gelu", residual=r, out=y) is y
    z, mag = product(x, W, b, r)
    want = act(z, "gelu")[0]
    within(y, want, act_bound(z, dense_bound(mag, K, dtype), "gelu") + want.abs() * half(dtype) * 1.01 + 2.0 ** -133)
    y.copy_(before[:, K + 2 * gap + N:K + 2 * gap + 2 * N])
    assert torch.equal(buf, before)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_backward(gpu, M, K, N, dtype):
    """dx beside x, and dW beside W, through the C entry point."""
    lib, dt, g = _lib.lib(), 1 if dtype == torch.bfloat16 else 0, gen(M)
    xs, ws = (torch.full((n, 2 * K + 1), 7.0, device="cuda", dtype=dtype) for n in (M, N))
    xs[:, :K], ws[:, :K] = rows(M, K, dtype, g), rows(N, K, dtype, g, N ** -0.5)
    dy = rows(M, N, dtype, g, 0.1)
    dx, dW, db, _ = dense.linear_backward(dy, xs[:, :K], ws[:, :K])
    n = C.c_size_t()
    assert lib.nflow_dense_linear_backward_workspace(M, N, K, dt, 1, C.byref(n)) == _lib.OK
    scratch = torch.empty(n.value + 16, device="cuda", dtype=torch.uint8)
    rc = lib.nflow_dense_linear_backward(dy.data_ptr(), dt, M, N, N, xs.data_ptr(), 2 * K + 1, ws.data_ptr(), 2 * K + 1, K, 0,
                                         None, N, None, N, xs[:, K:].data_ptr(), 2 * K + 1, ws[:, K:].data_ptr(), 2 * K + 1, None,
                                         scratch.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.OK, lib.nflow_last_error()
    torch.cuda.synchronize()
    assert torch.equal(xs[:, K:2 * K], dx) and torch.equal(ws[:, K:2 * K], dW)
    assert bool((xs[:, 2 * K] == 7).all()) and bool((ws[:, 2 * K] == 7).all())
