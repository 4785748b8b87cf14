"""Which kernel a block-FP8 product takes, as the library says without a GPU
(it then counts 256 CUs): the table that the GPU tests go by stays true."""
import ctypes as C

import pytest
import torch

from block_cuts import CUTS
from neuroflow_amd import _lib


def cut(M, N, K, out):
    edge, splits = C.c_int(-1), C.c_int(-1)
    assert _lib.lib().nflow_debug_fp8_block_cut(M, N, K, out, C.byref(edge), C.byref(splits)) == _lib.OK
    return edge.value, splits.value


@pytest.mark.skipif(torch.cuda.is_available(), reason="counts this GPU's CUs then")
@pytest.mark.parametrize("M,N,K,out,edge,splits", CUTS)
def test_cut(M, N, K, out, edge, splits):
    assert cut(M, N, K, out) == (edge, splits)


def test_every_kernel_has_a_size():
    assert {(e, out) for _, _, _, out, e, _ in CUTS} == {(0, 0), (0, 1), (64, 0), (64, 1), (128, 0), (128, 1), (256, 1)}
    large = [c for c in CUTS if c[4] == 256]
    assert any(c[2] % 256 > 0 and -(-c[2] // 128) % 2 == 1 and -(-c[2] // 128) >= 5 and c[0] % 256 and c[1] % 256 for c in large)


def test_refusals():
    e, s, lib = C.c_int(), C.c_int(), _lib.lib()
    for f in (lib.nflow_debug_fp8_block_cut, lib.nflow_debug_fp8_block_linear_kernel):
        assert f(-1, 8, 8, 0, C.byref(e), C.byref(s)) == _lib.INVALID_ARG
        assert f(8, 8, 8, 2, C.byref(e), C.byref(s)) == _lib.INVALID_ARG
        assert f(8, 8, 8, 0, None, C.byref(s)) == _lib.INVALID_ARG
        assert f(8, 8, 8, 0, C.byref(e), None) == _lib.INVALID_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="counts this GPU's CUs then")
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("M,N,K", [(17, 8192, 64), (17, 16384, 128), (17, 65536, 64), (24, 131072, 128), (33, 100000, 100),
                                   (64, 32768, 128), (65, 32768, 128), (65, 64000, 256), (128, 32768, 256),
                                   (200, 20000, 256), (1000, 4096, 128), (2000, 2048, 256)])
def test_few_rows_of_a_wide_layer_fill_the_chip(M, N, K, dtype):
    """The one-launch linear of many columns: its workgroups come to half the CUs
    at least wherever there is work for them (64 rows by 128 columns each)."""
    kernel, workgroups = C.c_int(-1), C.c_int(-1)
    assert _lib.lib().nflow_debug_fp8_block_linear_kernel(M, N, K, dtype, C.byref(kernel), C.byref(workgroups)) == _lib.OK
    if kernel.value == 1:
        assert 2 * workgroups.value >= min(256, -(-M // 64) * -(-N // 128))
