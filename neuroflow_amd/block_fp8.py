"""The linear layer in FP8 with a scale for every 128 values
(include/nflow_block.h): activations in 1 x 128 blocks, weights in 128 x 128
blocks, forward and backward.

Activations are float32 or bfloat16 CUDA tensors, contiguous (leading axes
are rows) or 2-D with a contiguous last axis and any row stride.  Results in
float32 come from bf16 matrix instructions on the codes' exact values, to fp32
accuracy; results in bfloat16 from FP8 ones, whose sums of 128 products are off
by up to 2^-12 of the products' magnitudes (1.3e-5 of the result on normal data;
more than its rounding only where products cancel).  A call runs on the current
stream of the current device, on which all of its tensors have to be; scratch
comes from torch's allocator.  A wrong type raises TypeError, a wrong shape or
device ValueError, a status of the library NflowError.  Nothing records an
autograd graph: results require no gradient whatever the inputs do, and
linear_backward is the caller's to call.
"""
from __future__ import annotations

import ctypes
import importlib.util
import sysconfig
from pathlib import Path
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .quant import _act

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_LIB_DIR = Path(__file__).resolve().parent / "lib"
_module = None


def _ops():
    """The built module block_ops (neuroflow_amd/bindings/block_ops.cpp), its
    calls bound to the library that is loaded."""
    global _module
    if _module is None:
        lib = _lib.lib()
        path = _LIB_DIR / ("block_ops" + sysconfig.get_config_var("EXT_SUFFIX"))
        if not path.exists():
            raise ImportError(f"{path} is not built; run `python -m neuroflow_amd.build` (there is no CPU fallback)")
        spec = importlib.util.spec_from_file_location("block_ops", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.bind(lambda name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value)
        _module = module
    return _module


class BlockFp8(NamedTuple):
    """A matrix of k columns in block FP8: codes (rows, 128 * ceil(k / 128))
    uint8 E4M3 bytes, zero past k; scales float32 (ceil(k / 128), rows), or for
    a weight (ceil(k / 128), ceil(rows / 128))."""

    codes: torch.Tensor
    scales: torch.Tensor
    k: int


# ---- quantise --------------------------------------------------------------------

def quantise(x: torch.Tensor) -> BlockFp8:
    """The rows of x (..., K) as block FP8."""
    c, s, k, _, _, _ = _ops().quantise(x, True, False)
    return BlockFp8(c, s, k)


def quantise_columns(x: torch.Tensor) -> BlockFp8:
    """The columns of x (M, K) as block FP8: K rows of M codes, what x^T is in
    a product over M."""
    _, _, _, c, s, k = _ops().quantise(x, False, True)
    return BlockFp8(c, s, k)


def quantise_both(x: torch.Tensor) -> Tuple[BlockFp8, BlockFp8]:
    """(quantise(x), quantise_columns(x)) from one read of x: what a training
    step keeps of an activation."""
    c, s, k, ct, st, kt = _ops().quantise(x, True, True)
    return BlockFp8(c, s, k), BlockFp8(ct, st, kt)


def quantise_weight(W: torch.Tensor, transposed: bool = False):
    """A weight (N, K) in 128 x 128 blocks; with transposed=True also the same
    codes as (K, N), for linear_backward."""
    c, s, k, ct, st, kt = _ops().quantise_weight(W, transposed)
    return (BlockFp8(c, s, k), BlockFp8(ct, st, kt)) if transposed else BlockFp8(c, s, k)


# ---- products ------------------------------------------------------------------------

def matmul(a: BlockFp8, w: BlockFp8, bias: Optional[torch.Tensor] = None, activation=None,
           out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """act(a w^T + bias), (rows of a, rows of w): a in 1 x 128 blocks, w in
    those or in 128 x 128 blocks."""
    if out_dtype not in _DTYPES:
        raise TypeError(f"out_dtype must be float32 or bfloat16, got {out_dtype}")
    return _ops().matmul(*a, *w, bias, _act(activation), _DTYPES[out_dtype])


def linear(x: torch.Tensor, w: BlockFp8, bias: Optional[torch.Tensor] = None, activation=None) -> torch.Tensor:
    """act(q(x) w^T + bias) in x's type: x (..., K) quantised in 1 x 128 blocks
    on the way, w a weight in 128 x 128 blocks."""
    return _ops().linear(x, *w, bias, _act(activation))


def linear_backward(dy: torch.Tensor, x_columns: BlockFp8, w_transposed: BlockFp8):
    """(dx, dW, dbias) of y = q(x) w^T + bias from dy (..., N): x_columns is
    quantise_columns(x) (or quantise_both's second), w_transposed
    quantise_weight's second.  dx has dy's shape and type, dW (N, K) and dbias
    (N) are float32; the quantise passes its gradient straight through."""
    return _ops().linear_backward(dy, *x_columns, *w_transposed)
