"""Operands on different GPUs are refused before anything is allocated or
launched.  Fake tensors carry a device and no memory, so no GPU is needed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from neuroflow_amd import block_fp8 as B
from neuroflow_amd import norm as L

M, N, K = 4, 200, 256


def _e(shape, dev, dtype=torch.float32):
    with FakeTensorMode():
        return torch.empty(shape, device=f"cuda:{dev}", dtype=dtype)


def _q(rows, k, codes=0, scales=0, weight=False):
    return B.BlockFp8(_e((rows, 128 * -(-k // 128)), codes, torch.uint8),
                      _e((-(-k // 128), -(-rows // 128) if weight else rows), scales), k)


def _x(dev=0, cols=K):
    return _e((M, cols), dev)


CALLS = {
    "layer_norm weight": lambda: L.layer_norm(_x(), _e(K, 1)),
    "layer_norm bias": lambda: L.layer_norm(_x(), None, _e(K, 1)),
    "layer_norm out": lambda: L.layer_norm(_x(), out=_x(1)),
    "layer_norm_fp8 weight": lambda: L.layer_norm_fp8(_x(), _e(K, 1)),
    "layer_norm_fp8 bias": lambda: L.layer_norm_fp8(_x(), _e(K, 0), _e(K, 1)),
    "layer_norm_backward dy": lambda: L.layer_norm_backward(_x(1), _x(), None, _e(M, 0), _e(M, 0)),
    "layer_norm_backward weight": lambda: L.layer_norm_backward(_x(), _x(), _e(K, 1), _e(M, 0), _e(M, 0)),
    "layer_norm_backward mean": lambda: L.layer_norm_backward(_x(), _x(), None, _e(M, 1), _e(M, 0)),
    "layer_norm_backward rstd": lambda: L.layer_norm_backward(_x(), _x(), None, _e(M, 0), _e(M, 1)),
    "matmul a.scales": lambda: B.matmul(_q(M, K, 0, 1), _q(N, K, weight=True)),
    "matmul w.codes": lambda: B.matmul(_q(M, K), _q(N, K, 1, 0, True)),
    "matmul w.scales": lambda: B.matmul(_q(M, K), _q(N, K, 0, 1, True)),
    "matmul w": lambda: B.matmul(_q(M, K), _q(N, K, 1, 1)),
    "matmul bias": lambda: B.matmul(_q(M, K), _q(N, K, weight=True), _e(N, 1)),
    "linear w.codes": lambda: B.linear(_x(), _q(N, K, 1, 0, True)),
    "linear w.scales": lambda: B.linear(_x(), _q(N, K, 0, 1, True)),
    "linear bias": lambda: B.linear(_x(), _q(N, K, weight=True), _e(N, 1)),
    "linear_backward x.codes": lambda: B.linear_backward(_x(0, N), _q(K, M, 1, 0), _q(K, N, weight=True)),
    "linear_backward x.scales": lambda: B.linear_backward(_x(0, N), _q(K, M, 0, 1), _q(K, N, weight=True)),
    "linear_backward w.codes": lambda: B.linear_backward(_x(0, N), _q(K, M), _q(K, N, 1, 0, True)),
    "linear_backward w.scales": lambda: B.linear_backward(_x(0, N), _q(K, M), _q(K, N, 0, 1, True)),
}


@pytest.mark.parametrize("name", CALLS)
def test_another_device_is_refused(name):
    with pytest.raises(ValueError, match="device|cuda:1"):
        CALLS[name]()
