"""The linear layer in FP8 with a scale for every 128 values
(include/nflow_block.h): activations in 1 x 128 blocks, weights in 128 x 128
blocks, forward and backward.

Activations are float32 or bfloat16 CUDA tensors whose last axis is
contiguous (leading axes are rows; a 2-D tensor may have any row stride).
Results in float32 come from bf16 matrix instructions on the codes' exact
values, results in bfloat16 from FP8 ones.  Calls run on the current stream;
scratch comes from torch's allocator.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import check
from .quant import _act, _p

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


class BlockFp8(NamedTuple):
    """A matrix of k columns in block FP8: codes (rows, 128 * ceil(k / 128))
    uint8 E4M3 bytes, zero past k; scales float32 (ceil(k / 128), rows), or for
    a weight (ceil(k / 128), ceil(rows / 128))."""

    codes: torch.Tensor
    scales: torch.Tensor
    k: int


# ---- arguments -----------------------------------------------------------------

def _dtype(t: torch.Tensor) -> int:
    return _DTYPES[t.dtype]


def _activation(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}, "
                         f"got {tuple(t.shape)} {t.dtype} on {t.device}")
    return t


def _matrix(t: torch.Tensor, name: str) -> Tuple[int, int, int]:
    """(rows, columns, row stride) of an activation."""
    _activation(t, name)
    shape = t.shape
    if len(shape) == 0:
        raise ValueError(f"{name} needs an axis")
    K = shape[-1]
    if t.is_contiguous():
        return (shape[0] if len(shape) == 2 else math.prod(shape[:-1])), K, K
    if t.dim() > 2 or t.stride(-1) != 1 or t.stride(0) < K:
        raise ValueError(f"{name} must be contiguous, or 2-D with a contiguous last axis")
    return t.shape[0], K, t.stride(0)


def _param(t: Optional[torch.Tensor], n: int, name: str, required: bool = False) -> None:
    if t is None:
        if required:
            raise TypeError(f"{name} is required")
        return
    if type(t) is torch.Tensor and t.dtype is torch.float32 and t.is_cuda and t.shape == (n,) and t.is_contiguous():
        return
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be torch.float32, got {t.dtype}")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be {n} contiguous values, got {tuple(t.shape)}")


def _block(q: BlockFp8, name: str, weight: bool = False) -> int:
    """Rows of q, whose scales are a weight's (128 x 128 blocks) or not."""
    codes, scales, k = q
    kb = (k + 127) >> 7
    if not codes.is_cuda or not scales.is_cuda:
        raise TypeError(f"{name} must hold CUDA tensors")
    if codes.dtype != torch.uint8 or scales.dtype != torch.float32:
        raise TypeError(f"{name} must hold uint8 codes and float32 scales")
    if codes.dim() != 2 or codes.shape[1] != 128 * kb or not codes.is_contiguous():
        raise ValueError(f"{name}.codes must be a contiguous (rows, {128 * kb}) for k = {k}, got {tuple(codes.shape)}")
    R = codes.shape[0]
    if not scales.is_contiguous() or scales.shape != (kb, (R + 127) >> 7 if weight else R):
        raise ValueError(f"{name}.scales must be a contiguous ({kb}, {(R + 127) >> 7 if weight else R}), "
                         f"got {tuple(scales.shape)}")
    return R


def _is_weight(q: BlockFp8) -> bool:
    return q.scales.dim() == 2 and q.scales.shape[1] != q.codes.shape[0]


def _empty_block(R: int, K: int, device) -> BlockFp8:
    kb = (K + 127) >> 7
    return BlockFp8(torch.empty(R, 128 * kb, dtype=torch.uint8, device=device),
                    torch.empty(kb, R, dtype=torch.float32, device=device), K)


def _stream(t: torch.Tensor) -> int:
    """The current stream's handle, on t's device, which has to be the current one."""
    i = t.get_device()
    if i != torch._C._cuda_getDevice():
        raise ValueError(f"the tensors are on cuda:{i}, the current device is cuda:{torch._C._cuda_getDevice()}")
    return torch._C._cuda_getCurrentRawStream(i)


def _workspace(n: int, device) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


# ---- quantise --------------------------------------------------------------------

def quantise(x: torch.Tensor) -> BlockFp8:
    """The rows of x (..., K) as block FP8."""
    M, K, ldx = _matrix(x, "x")
    q = _empty_block(M, K, x.device)
    check(_lib.lib().nflow_fp8_block_quantise(_p(x), _dtype(x), M, K, ldx, _p(q.codes), _p(q.scales), None, None,
                                              _stream(x)), "fp8_block_quantise")
    return q


def quantise_columns(x: torch.Tensor) -> BlockFp8:
    """The columns of x (M, K) as block FP8: K rows of M codes, what x^T is in
    a product over M."""
    M, K, ldx = _matrix(x, "x")
    t = _empty_block(K, M, x.device)
    check(_lib.lib().nflow_fp8_block_quantise(_p(x), _dtype(x), M, K, ldx, None, None, _p(t.codes), _p(t.scales),
                                              _stream(x)), "fp8_block_quantise")
    return t


def quantise_both(x: torch.Tensor) -> Tuple[BlockFp8, BlockFp8]:
    """(quantise(x), quantise_columns(x)) from one read of x: what a training
    step keeps of an activation."""
    M, K, ldx = _matrix(x, "x")
    q, t = _empty_block(M, K, x.device), _empty_block(K, M, x.device)
    check(_lib.lib().nflow_fp8_block_quantise(_p(x), _dtype(x), M, K, ldx, _p(q.codes), _p(q.scales), _p(t.codes),
                                              _p(t.scales), _stream(x)), "fp8_block_quantise")
    return q, t


def quantise_weight(W: torch.Tensor, transposed: bool = False):
    """A weight (N, K) in 128 x 128 blocks; with transposed=True also the same
    codes as (K, N), for linear_backward."""
    N, K, ldw = _matrix(W, "W")
    nb, kb = (N + 127) >> 7, (K + 127) >> 7
    w = BlockFp8(torch.empty(N, 128 * kb, dtype=torch.uint8, device=W.device),
                 torch.empty(kb, nb, dtype=torch.float32, device=W.device), K)
    t = None
    if transposed:
        t = BlockFp8(torch.empty(K, 128 * nb, dtype=torch.uint8, device=W.device),
                     torch.empty(nb, kb, dtype=torch.float32, device=W.device), N)
    check(_lib.lib().nflow_fp8_block_quantise_weight(_p(W), _dtype(W), N, K, ldw, _p(w.codes), _p(w.scales),
                                                     _p(t.codes) if t else None, _p(t.scales) if t else None,
                                                     _stream(W)), "fp8_block_quantise_weight")
    return (w, t) if transposed else w


# ---- products ------------------------------------------------------------------------

def matmul(a: BlockFp8, w: BlockFp8, bias: Optional[torch.Tensor] = None, activation=None,
           out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """act(a w^T + bias), (rows of a, rows of w): a in 1 x 128 blocks, w in
    those or in 128 x 128 blocks."""
    if a.k != w.k:
        raise ValueError(f"a has {a.k} columns, w has {w.k}")
    if out_dtype not in _DTYPES:
        raise TypeError(f"out_dtype must be float32 or bfloat16, got {out_dtype}")
    M = _block(a, "a")
    blocks = _is_weight(w)
    N = _block(w, "w", weight=blocks)
    _param(bias, N, "bias")
    out = torch.empty(M, N, dtype=out_dtype, device=a.codes.device)
    L, dt = _lib.lib(), _DTYPES[out_dtype]
    n = C.c_size_t()
    check(L.nflow_fp8_block_matmul_workspace(M, N, a.k, dt, C.byref(n)), "fp8_block_matmul")
    ws = _workspace(n.value, out.device)
    check(L.nflow_fp8_block_matmul(_p(a.codes), _p(a.scales), _p(w.codes), _p(w.scales), int(blocks), M, N, a.k,
                                   _p(bias), _act(activation), _p(out), dt, N, _p(ws), n.value, _stream(out)),
          "fp8_block_matmul")
    return out


def linear(x: torch.Tensor, w: BlockFp8, bias: Optional[torch.Tensor] = None, activation=None) -> torch.Tensor:
    """act(q(x) w^T + bias) in x's type: x (..., K) quantised in 1 x 128 blocks
    on the way, w a weight in 128 x 128 blocks."""
    M, K, ldx = _matrix(x, "x")
    if w.k != K:
        raise ValueError(f"x has {K} columns, w has {w.k}")
    N = _block(w, "w", weight=True)
    _param(bias, N, "bias")
    y = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=x.device)
    L, dt = _lib.lib(), _dtype(x)
    n = C.c_size_t()
    check(L.nflow_fp8_block_linear_workspace(M, N, K, dt, C.byref(n)), "fp8_block_linear")
    ws = _workspace(n.value, x.device)
    check(L.nflow_fp8_block_linear(_p(x), dt, M, K, ldx, _p(w.codes), _p(w.scales), N, _p(bias), _act(activation),
                                   _p(y), N, _p(ws), n.value, _stream(x)), "fp8_block_linear")
    return y


def linear_backward(dy: torch.Tensor, x_columns: BlockFp8, w_transposed: BlockFp8):
    """(dx, dW, dbias) of y = q(x) w^T + bias from dy (..., N): x_columns is
    quantise_columns(x) (or quantise_both's second), w_transposed
    quantise_weight's second.  dx has dy's shape and type, dW (N, K) and dbias
    (N) are float32; the quantise passes its gradient straight through."""
    M, N, lddy = _matrix(dy, "dy")
    K = _block(w_transposed, "w_transposed", weight=True)
    if w_transposed.k != N:
        raise ValueError(f"dy has {N} columns, w_transposed has {w_transposed.k}")
    if x_columns.k != M or _block(x_columns, "x_columns") != K:
        raise ValueError(f"x_columns must be ({K} rows, k = {M}), got ({x_columns.codes.shape[0]}, {x_columns.k})")
    dx = torch.empty(*dy.shape[:-1], K, dtype=dy.dtype, device=dy.device)
    dW = torch.empty(N, K, dtype=torch.float32, device=dy.device)
    db = torch.empty(N, dtype=torch.float32, device=dy.device)
    L, dt = _lib.lib(), _dtype(dy)
    n = C.c_size_t()
    check(L.nflow_fp8_block_linear_backward_workspace(M, N, K, dt, C.byref(n)), "fp8_block_linear_backward")
    ws = _workspace(n.value, dy.device)
    check(L.nflow_fp8_block_linear_backward(_p(dy), dt, M, N, lddy, _p(x_columns.codes), _p(x_columns.scales),
                                            _p(w_transposed.codes), _p(w_transposed.scales), K, _p(dx), K, _p(dW),
                                            _p(db), _p(ws), n.value, _stream(dy)), "fp8_block_linear_backward")
    return dx, dW, db
