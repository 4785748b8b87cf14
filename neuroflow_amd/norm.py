"""Layer norm over the last axis of an activation, forward and backward, and
straight into 128-block FP8 (include/nflow_block.h).

The norm is the one ahead of a token mixer's projections
(cpp/src/fno.cpp:1418-1438).  Activations are float32 or bfloat16 CUDA
tensors whose last axis is contiguous; parameters and their gradients are
float32.  Calls run on the current stream.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from ._lib import check
from .block_fp8 import _activation, _dtype, _empty_block, _matrix, _param, _stream, _workspace
from .quant import _p


def _params(D: int, weight, bias) -> None:
    _param(weight, D, "weight")
    _param(bias, D, "bias")


def _stats(M: int, like: torch.Tensor, wanted: bool):
    if not wanted:
        return None, None
    mean = torch.empty(M, dtype=torch.float32, device=like.device)
    return mean, torch.empty_like(mean)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out: Optional[torch.Tensor] = None, return_stats: bool = False):
    """(x - mean) * rstd * weight + bias over the last axis; with
    return_stats also the fp32 mean and rstd of every row, which the backward
    pass takes.  out may be x."""
    M, D, ldx = _matrix(x, "x")
    _params(D, weight, bias)
    if out is None:
        y, ldy = torch.empty_like(x, memory_format=torch.contiguous_format), D
    else:
        y, ldy = out, _matrix(_activation(out, "out", like=x), "out")[2]
    mean, rstd = _stats(M, x, return_stats)
    check(_lib.lib().nflow_layer_norm_forward(_p(x), _dtype(x), M, D, ldx, _p(weight), _p(bias), float(eps), _p(y),
                                              ldy, _p(mean), _p(rstd), _stream(x)), "layer_norm")
    return (y, mean, rstd) if return_stats else y


def layer_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-5, return_stats: bool = False):
    """layer_norm as the next product takes it: block-FP8 codes and scales of
    the rows, quantised from the fp32 result."""
    M, D, ldx = _matrix(x, "x")
    _params(D, weight, bias)
    q = _empty_block(M, D, x.device)
    mean, rstd = _stats(M, x, return_stats)
    check(_lib.lib().nflow_layer_norm_fp8_block(_p(x), _dtype(x), M, D, ldx, _p(weight), _p(bias), float(eps),
                                                _p(q.codes), _p(q.scales), _p(mean), _p(rstd), _stream(x)),
          "layer_norm_fp8")
    return (q, mean, rstd) if return_stats else q


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor):
    """(dx, dweight, dbias) from the mean and rstd of the forward pass.  The
    gradients of the parameters are fp32 sums over all rows, in an order that
    does not change from call to call; weight None stands for ones."""
    M, D, ldx = _matrix(x, "x")
    _activation(dy, "dy", like=x)
    lddy = _matrix(dy, "dy")[2]
    _param(weight, D, "weight")
    _param(mean, M, "mean", required=True)
    _param(rstd, M, "rstd", required=True)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty(2, D, dtype=torch.float32, device=x.device)
    L = _lib.lib()
    n = C.c_size_t()
    check(L.nflow_layer_norm_backward_workspace(M, D, C.byref(n)), "layer_norm_backward")
    ws = _workspace(n.value, x.device)
    check(L.nflow_layer_norm_backward(_p(dy), _p(x), _dtype(x), M, D, lddy, ldx, _p(weight), _p(mean), _p(rstd),
                                      _p(dx), D, _p(dw), dw.data_ptr() + 4 * D, _p(ws), n.value, _stream(x)),
          "layer_norm_backward")
    return dx, dw[0], dw[1]
