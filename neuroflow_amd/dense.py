"""The linear layer in bfloat16 or float32, with bias, residual and activation in
the product's epilogue, forward and backward (include/nflow_residual.h).

For the layers of a model that stay unquantised beside quant's and block_fp8's.
x, W, the residual and the results are CUDA tensors of one type; x, the residual
and dy are contiguous (leading axes are rows) or 2-D with a contiguous last axis
and any row stride, W is (N, K).  bias and its gradient are float32.  Sums are
fp32; float32 products are formed from three bfloat16 parts of each operand, to
fp32 accuracy (an infinite operand gives NaN there, with ReLU too, and one below
2^-110 is held to 2^-134).  bfloat16 operands whose rows are not whole 16-byte groups
are copied to scratch at every call, but for some of few rows.  A call runs on the
current stream of the current device, on which all of its tensors have to be; scratch
comes from torch's allocator.  A wrong type raises TypeError, a wrong shape or
device ValueError, a status of the library NflowError.  Nothing records an
autograd graph: results require no gradient whatever the inputs do, and
linear_backward is the caller's to call.
"""
from __future__ import annotations

from typing import Optional

import torch

from .block_fp8 import _ops
from .quant import _act


def linear(x: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor] = None, activation=None,
           residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, return_pre: bool = False):
    """act(x W^T + bias + residual).  The residual joins ahead of the
    activation, as in quant's layers; out may be the residual (a stream updated
    in place), but share no other memory with an input (columns of one buffer
    share none).  With return_pre also what the activation was applied to, in x's
    type, which linear_backward takes."""
    y, pre = _ops().dense_linear(x, W, bias, _act(activation), residual, out, return_pre)
    return (y, pre) if return_pre else y


def linear_backward(dy: torch.Tensor, x: torch.Tensor, W: torch.Tensor, activation=None,
                    pre: Optional[torch.Tensor] = None):
    """(dx, dW, dbias, dz) of linear from dy (..., N): dz = dy act'(pre) is the
    gradient of the residual too, and dy itself with no activation.  pre is what
    linear returned with return_pre (for ReLU its result serves as well).  dx,
    dW and dz have dy's type, and the products take dz as it is returned, in
    bfloat16 rounded a first time; dbias is float32, summed ahead of that rounding."""
    return _ops().dense_linear_backward(dy, x, W, _act(activation), pre)
