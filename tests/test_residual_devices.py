"""Operands on different GPUs are refused before anything is allocated or
launched.  Fake tensors carry a device and no memory, so no GPU is needed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from neuroflow_amd import dense, grads
from neuroflow_amd import norm as L

M, N, K = 40, 24, 64


def _e(shape, dev=0):
    with FakeTensorMode():
        return torch.empty(shape, device=f"cuda:{dev}")


X, W, R = (M, K), (N, K), (M, N)
CALLS = {
    "rms_norm weight": lambda: L.rms_norm(_e(X), _e(K, 1)),
    "rms_norm residual": lambda: L.rms_norm(_e(X), residual=_e(X, 1)),
    "rms_norm sum_out": lambda: L.rms_norm(_e(X), residual=_e(X), sum_out=_e(X, 1)),
    "rms_norm_fp8 weight": lambda: L.rms_norm_fp8(_e(X), _e(K, 1)),
    "rms_norm_fp8 residual": lambda: L.rms_norm_fp8(_e(X), residual=_e(X, 1)),
    "rms_norm_backward dy": lambda: L.rms_norm_backward(_e(X, 1), _e(X), None, _e(M)),
    "rms_norm_backward weight": lambda: L.rms_norm_backward(_e(X), _e(X), _e(K, 1), _e(M)),
    "rms_norm_backward rstd": lambda: L.rms_norm_backward(_e(X), _e(X), None, _e(M, 1)),
    "rms_norm_backward dsum": lambda: L.rms_norm_backward(_e(X), _e(X), None, _e(M), dsum=_e(X, 1)),
    "linear W": lambda: dense.linear(_e(X), _e(W, 1)),
    "linear bias": lambda: dense.linear(_e(X), _e(W), _e(N, 1)),
    "linear residual": lambda: dense.linear(_e(X), _e(W), residual=_e(R, 1)),
    "linear out": lambda: dense.linear(_e(X), _e(W), out=_e(R, 1)),
    "linear_backward x": lambda: dense.linear_backward(_e(R), _e(X, 1), _e(W)),
    "linear_backward W": lambda: dense.linear_backward(_e(R), _e(X), _e(W, 1)),
    "linear_backward pre": lambda: dense.linear_backward(_e(R), _e(X), _e(W), "gelu", pre=_e(R, 1)),
    "global_norm": lambda: grads.global_norm([_e(X), _e(X, 1)]),
    "clip gradient": lambda: grads.clip_by_global_norm([_e(X), _e(X, 1)], 1.0),
    "clip out": lambda: grads.clip_by_global_norm([_e(X)], 1.0, out=[_e(X, 1)]),
}


@pytest.mark.parametrize("name", CALLS)
def test_another_device_is_refused(name):
    if torch.cuda.is_available() and torch.cuda.device_count() < 2:
        pytest.skip("the second device has to exist where one does")
    with pytest.raises(ValueError, match="device|cuda:1"):
        CALLS[name]()
