"""The bf16 linear layer of few rows whose operands the tiles would have to copy: the
kernel that a call takes goes by how its rows lie, and the room asked for by that too."""
import ctypes as C

import pytest
import torch

from neuroflow_amd import _lib, dense
from residual_reference import half, rows, gen, within
from residual_reference import dense as product, dense_bound


def room(M, K, N, copies):
    n = C.c_size_t()
    assert _lib.lib().nflow_dense_linear_workspace(M, N, K, 1, copies, C.byref(n)) == _lib.OK
    return n.value


ANY, WORDS = 1, 2


@pytest.mark.parametrize("M,K,N", [(17, 16382, 16384), (24, 4094, 16384), (32, 4094, 1024), (16, 8190, 8192), (1, 1022, 16384)])
def test_no_copies_of_words(M, K, N):
    """Rows at whole words: the weight is read in place, where copies of it cost up to twice the
    call.  (There may be room for x's, beside a weight that needs none.)"""
    assert room(M, K, N, WORDS) < 2 * N * K


@pytest.mark.parametrize("M,K,N", [(1, 1023, 16384), (1, 16383, 16384), (8, 8191, 4096), (16, 1023, 4096)])
def test_no_copies_of_few_odd_rows(M, K, N):
    assert room(M, K, N, ANY) < 2 * N * K


@pytest.mark.parametrize("M,K,N", [(17, 4095, 1024), (32, 8191, 4096), (24, 16383, 16384), (1, 16383, 256)])
def test_copies_of_odd_rows(M, K, N):
    """Rows at odd addresses, which hold the few-row kernel up more than their copies cost."""
    assert room(M, K, N, ANY) >= 2 * N * K


@pytest.mark.parametrize("M,K,N", [(1, 4096, 4096), (17, 4095, 1024), (32, 16382, 16384), (100, 2021, 1001), (33, 64, 64)])
def test_the_room_covers_every_lie(M, K, N):
    assert room(M, K, N, 0) <= room(M, K, N, WORDS) <= room(M, K, N, ANY)
    if M > 32:                     # tiles always: their copies however the rows lie
        assert room(M, K, N, WORDS) == room(M, K, N, ANY) >= 2 * K * (M + N)


def lying(n, K, how, g):
    """(n, K) rows in groups (as far as K is), in words, at odd strides, or at an odd address."""
    even = next(p for p in range(9) if (K + p) % 2 == 0 and ((K + p) % 8 or K % 8))
    pad, skip = {"groups": (-K % 8, 0), "words": (even, 0), "stride": (1 - K % 2, 0), "address": (-K % 8, 1)}[how]
    flat = torch.full((n * (K + pad) + 8,), float("nan"), device="cuda", dtype=torch.bfloat16)
    t = flat[skip:skip + n * (K + pad)].view(n, K + pad)[:, :K]
    t.copy_(rows(n, K, torch.bfloat16, g))
    return t


@pytest.mark.gpu
@pytest.mark.parametrize("K,N", [(7, 3), (1023, 300), (4094, 1024), (4096, 64), (4095, 4096), (8192, 100)])
@pytest.mark.parametrize("hx", ["groups", "words", "stride", "address"])
@pytest.mark.parametrize("hw", ["groups", "words", "stride", "address"])
def test_against_64_bits(gpu, K, N, hx, hw):
    g = gen(K)
    W = lying(N, K, hw, g)
    for M in (1, 16, 17, 32, 33):
        x = lying(M, K, hx, g)
        z, mag = product(x, W)
        within(dense.linear(x, W), z, dense_bound(mag, K, torch.bfloat16) + z.abs() * half(torch.bfloat16) * 1.01)
