"""The norm of many gradients together, and their clipping by it
(include/nflow_residual.h).

Gradients are contiguous float32 or bfloat16 CUDA tensors, mixed as they come,
on the current device; a call runs on its current stream and reads nothing back:
the norm is a tensor on the GPU.  A wrong type raises TypeError, a wrong shape or
device ValueError, a status of the library NflowError.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .block_fp8 import _ops


def global_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """The root of the sum of squares over all gradients, a float32 scalar;
    squares and sums are taken in 64 bits."""
    return _ops().global_norm(list(grads))


def clip_by_global_norm(grads: Sequence[torch.Tensor], max_norm: float,
                        out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Multiplies every gradient by min(1, max_norm / norm), in place or into the
    tensors of out, and returns the norm.  A NaN in any gradient makes all of them
    NaN, an infinity makes the finite ones 0: the norm, NaN or infinite, tells.  With
    an infinite max_norm and no NaN all are left as they are."""
    return _ops().clip_by_global_norm(list(grads), float(max_norm), None if out is None else list(out))
