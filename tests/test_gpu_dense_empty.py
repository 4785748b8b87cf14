"""The linear layer's gradients where a size is zero: sums over nothing are zeros,
written like any other result."""
import ctypes as C

import pytest
import torch

from neuroflow_amd import _lib, dense
from residual_reference import DTYPES, gen, rows

pytestmark = pytest.mark.gpu


def used(*size, dtype):
    """Leaves memory of this size that is not zero to the allocator's next tensor of it."""
    torch.full(size, float("nan"), device="cuda", dtype=dtype)


@pytest.mark.parametrize("kind", [None, "relu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (8, 64), (33, 70), (300, 513)])
def test_no_outputs(gpu, M, K, dtype, kind):
    """N = 0: dx is the sum over no columns."""
    x = rows(M, K, dtype, gen(1))
    dy, W = (torch.empty(s, device="cuda", dtype=dtype) for s in ((M, 0), (0, K)))
    used(M, K, dtype=dtype)
    dx, dW, db, dz = dense.linear_backward(dy, x, W, kind, pre=dy if kind else None)
    assert dx.shape == (M, K) and torch.equal(dx, torch.zeros_like(dx))
    assert dW.shape == (0, K) and db.shape == (0,) and dz.shape == (M, 0)


@pytest.mark.parametrize("kind", [None, "relu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1, 1), (8, 64), (33, 70), (300, 513)])
def test_no_inputs(gpu, M, N, dtype, kind):
    """K = 0: dz and dbias are what they are at any K."""
    dy, pre = rows(M, N, dtype, gen(2)), rows(M, N, dtype, gen(3)) if kind else None
    x, W = (torch.empty(s, device="cuda", dtype=dtype) for s in ((M, 0), (N, 0)))
    dx, dW, db, dz = dense.linear_backward(dy, x, W, kind, pre=pre)
    assert dx.shape == (M, 0) and dW.shape == (N, 0)
    want = dense.linear_backward(dy, torch.ones(M, 8, device="cuda", dtype=dtype), torch.ones(N, 8, device="cuda", dtype=dtype),
                                 kind, pre=pre)
    assert torch.equal(dz, want[3])
    total = dz.double().abs().sum(0) if kind is None else dy.double().abs().sum(0) * 1.13
    assert bool(((db.double() - want[2].double()).abs() <= total * 2 * (M + 8) * 2.0 ** -24).all())


@pytest.mark.parametrize("kind", [None, "gelu"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(gpu, dtype, kind):
    """M = 0: dW and dbias are sums over no rows."""
    x, W = rows(0, 70, dtype, gen(4)), rows(40, 70, dtype, gen(5))
    dy = rows(0, 40, dtype, gen(6))
    used(40, 70, dtype=dtype)
    used(40, dtype=torch.float32)
    dx, dW, db, dz = dense.linear_backward(dy, x, W, kind, pre=dy if kind else None)
    assert dx.shape == (0, 70) and dz.shape == (0, 40)
    assert torch.equal(dW, torch.zeros_like(W)) and torch.equal(db, torch.zeros(40, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_gradient_asked_for(gpu, dtype):
    """Each gradient by itself through the C entry point, at every size that may be zero."""
    lib, dt = _lib.lib(), 1 if dtype == torch.bfloat16 else 0
    for M, N, K in ((8, 0, 64), (0, 8, 64), (8, 8, 0), (8, 0, 0), (0, 0, 64), (8, 16, 64)):
        dy, x, W = rows(M, N, dtype, gen(7)), rows(M, K, dtype, gen(8)), rows(N, K, dtype, gen(9))
        n = C.c_size_t()
        assert lib.nflow_dense_linear_backward_workspace(M, N, K, dt, 1, C.byref(n)) == _lib.OK
        ws = torch.empty(n.value + 16, device="cuda", dtype=torch.uint8)
        want = (dy.double() @ W.double(), dy.double().t() @ x.double(), dy.double().sum(0))
        for which in range(3):
            out = torch.full(want[which].shape, float("nan"), device="cuda", dtype=torch.float32 if which == 2 else dtype)
            to = [out.data_ptr() if i == which else None for i in range(3)]
            rc = lib.nflow_dense_linear_backward(dy.data_ptr(), dt, M, N, N, x.data_ptr(), K, W.data_ptr(), K, K, 0, None, N, None, N,
                                                 to[0], K, to[1], K, to[2], ws.data_ptr(), n.value,
                                                 torch.cuda.current_stream().cuda_stream)
            assert rc == _lib.OK, (M, N, K, which)
            torch.cuda.synchronize()
            # Sums of at most 64 terms in fp32, and a rounding.
            most = 2.0 ** -8 if dtype == torch.bfloat16 and which < 2 else 2.0 ** -24
            terms = (dy.double().abs() @ W.double().abs(), dy.double().abs().t() @ x.double().abs(), dy.double().abs().sum(0))[which]
            assert bool(((out.double() - want[which]).abs() <= terms * (most + 2.0 ** -15)).all()), (M, N, K, which)
