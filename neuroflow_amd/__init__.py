"""neuroflow_amd -- NeuroFlow's quantised inference GEMM on AMD MI355X (gfx950).

The compute lives in libnflow_quant.so (hand-written HIP kernels behind the
C-ABI of include/nflow_quant.h); this package is its Python front-end:

  quant      the nflow-quant API (int8_gemm::*, the FP8 E4M3 codec) on
             torch CUDA tensors, plus Int8Linear / Fp8Linear layers
  norm       layer norm, and RMS norm with the residual's addition, forward
             (also straight to block FP8) and backward
  block_fp8  the linear layer in FP8 with a scale for every 128 values,
             forward and backward
  dense      the linear layer in bf16 or fp32 with bias, residual and
             activation in its epilogue, forward and backward
  grads      the norm of many gradients, and their clipping by it
  workloads  the seeded synthetic inputs of the benchmark configurations
  build      in-tree build of libnflow_quant.so
"""
from ._lib import NflowError, lib  # noqa: F401

__all__ = ["NflowError", "lib"]
