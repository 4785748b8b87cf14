"""Layer norm and RMS norm over the last axis of an activation, forward and
backward, and straight into 128-block FP8 (include/nflow_block.h,
include/nflow_residual.h).

The layer norm is the one ahead of a token mixer's projections
(cpp/src/fno.cpp:1418-1438); the RMS norm takes a residual's addition on its way.  Activations are float32 or bfloat16 CUDA
tensors, contiguous or 2-D with a contiguous last axis and any row stride;
parameters and their gradients are float32.  A call runs on the current stream
of the current device, on which all of its tensors have to be.  A wrong type
raises TypeError, a wrong shape or device ValueError, a status of the library
NflowError.  Nothing records an autograd graph: results require no gradient
whatever the inputs do, and the backward functions are the caller's to call.
"""
from __future__ import annotations

from typing import Optional

import torch

from .block_fp8 import BlockFp8, _ops


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out: Optional[torch.Tensor] = None, return_stats: bool = False):
    """(x - mean) * rstd * weight + bias over the last axis; with
    return_stats also the fp32 mean and rstd of every row, which the backward
    pass takes.  out may be x, but not overlap it otherwise."""
    return _ops().layer_norm(x, weight, bias, eps, out, return_stats)


def layer_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                   eps: float = 1e-5, return_stats: bool = False):
    """layer_norm as the next product takes it: block-FP8 codes and scales of
    the rows, quantised from the fp32 result."""
    codes, scales, k, mean, rstd = _ops().layer_norm_fp8(x, weight, bias, eps, return_stats)
    q = BlockFp8(codes, scales, k)
    return (q, mean, rstd) if return_stats else q


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor):
    """(dx, dweight, dbias) from the mean and rstd of the forward pass.  The
    gradients of the parameters are fp32 sums over all rows, in an order that
    does not change from call to call; weight None stands for ones."""
    return _ops().layer_norm_backward(dy, x, weight, mean, rstd)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
             residual: Optional[torch.Tensor] = None, sum_out: Optional[torch.Tensor] = None, return_stats: bool = False):
    """t * rstd * weight with t = x + residual and rstd = 1 / sqrt(mean(t^2) +
    eps) over the last axis.  Returns y; with a residual also t, rounded to x's
    type (the norm is of the unrounded one); with return_stats also the fp32
    rstd of every row, which the backward pass takes.  sum_out receives t and
    may be the residual or x, row for row: a stream updated in place."""
    y, total, rstd = _ops().rms_norm(x, weight, eps, residual, sum_out, return_stats)
    return _results(y, total if residual is not None else None, rstd)


def rms_norm_fp8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                 residual: Optional[torch.Tensor] = None, sum_out: Optional[torch.Tensor] = None,
                 return_stats: bool = False):
    """rms_norm as the next product takes it: y as block-FP8 codes and scales of
    the rows, quantised from the fp32 result."""
    codes, scales, k, total, rstd = _ops().rms_norm_fp8(x, weight, eps, residual, sum_out, return_stats)
    return _results(BlockFp8(codes, scales, k), total if residual is not None else None, rstd)


def rms_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], rstd: torch.Tensor,
                      dsum: Optional[torch.Tensor] = None):
    """(dx, dweight) from what was normed (x, or with a residual the sum that
    rms_norm returned) and the rstd of the forward pass.  dsum is the gradient
    that the sum has from its other use, the residual stream; it joins dx, which
    is then the gradient of the forward pass's x and residual alike.  dweight is
    an fp32 sum over all rows, in an order that does not change from call to
    call; weight None stands for ones."""
    return _ops().rms_norm_backward(dy, x, weight, rstd, dsum)


def _results(y, total, rstd):
    """y alone, or a tuple of those that were asked for."""
    rest = tuple(t for t in (total, rstd) if t is not None)
    return (y, *rest) if rest else y
