"""The error of block-FP8 products ahead of their last rounding, against the
bounds that include/nflow_block.h states."""
import pytest
import torch

from block_cuts import BF16, F32
from neuroflow_amd import block_fp8 as B

pytestmark = pytest.mark.gpu

TYPES = {F32: torch.float32, BF16: torch.bfloat16}

# One row many times over, and minus the exact result as the bias: the output is
# then the product's own error, as it stands before the last rounding.
ERRORS = [(1, 2000, 1024), (64, 2000, 1024), (300, 2000, 1024), (2000, 1900, 900), (4090, 4000, 600), (20, 3000, 200),
          (300, 2000, 8192)]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M,N,K", ERRORS)
def test_error_before_rounding(gpu, M, N, K, out):
    """Normal operands: 1.3e-5 of the result in the 2-norm by the FP8
    instruction (a half as much again allowed for the draw), and for an fp32
    result 1e-7 by the bf16 one and at most 2 blocks + 4 roundings of 2^-24 in
    random directions, of sums no larger than a few results."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a = B.quantise(torch.randn(1, K, generator=g, device="cuda"))
    w = B.quantise_weight(torch.randn(N, K, generator=g, device="cuda") / K ** 0.5)
    av = a.codes.view(torch.float8_e4m3fn).float().double().view(-1, 128) * a.scales.double().view(-1, 1)
    s = w.scales.double().t().repeat_interleave(128, 0)[:N]
    wv = w.codes.view(torch.float8_e4m3fn).float().double().view(N, -1, 128) * s[:, :, None]
    terms = wv * av
    exact, blocks = terms.sum((1, 2)), terms.abs().sum((1, 2))
    rows = B.BlockFp8(a.codes.repeat(M, 1), a.scales.repeat(1, M), K)
    err = B.matmul(rows, w, -exact.float(), out_dtype=TYPES[out]).double()
    assert torch.equal(err, err[:1].expand(M, N))
    err = err[0] - (exact - exact.float().double())
    rel = float(err.norm() / exact.norm())
    assert rel <= (2e-5 if out == BF16 else 1e-7 + 2.0 ** -24 * 3 * (2 * -(-K // 128) + 4) ** 0.5), rel
    # And at no result more than the documented part of the magnitudes (or 128 + 2 blocks + 4 roundings for fp32).
    bound = blocks * (2.0 ** -12 if out == BF16 else (128 + 2 * -(-K // 128) + 4) * 2.0 ** -24)
    assert (err.abs() <= bound).all(), float((err.abs() / bound).max())


@pytest.mark.parametrize("M", [1, 64, 300, 4090])
def test_error_under_cancellation(gpu, M):
    """Products that cancel to a thousandth of their magnitudes, in bf16: the
    error stays below 2^-12 of the magnitudes, which is not below bf16's
    rounding of what is left."""
    N, K = 4000, 640
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(1, K // 2, generator=g, device="cuda")
    W = torch.randn(N, K // 2, generator=g, device="cuda")
    W2 = -W * (1 + 2e-3 * torch.randn(N, K // 2, generator=g, device="cuda"))

    def pairs(p, q):                    # neighbouring columns cancel, within one K block
        return torch.stack((p, q), 2).flatten(1)

    a, w = B.quantise(pairs(x, x)), B.quantise_weight(pairs(W, W2))
    av = a.codes.view(torch.float8_e4m3fn).float().double().view(-1, 128) * a.scales.double().view(-1, 1)
    s = w.scales.double().t().repeat_interleave(128, 0)[:N]
    terms = w.codes.view(torch.float8_e4m3fn).float().double().view(N, -1, 128) * s[:, :, None] * av
    exact, mag = terms.sum((1, 2)), terms.abs().sum((1, 2))
    rows = B.BlockFp8(a.codes.repeat(M, 1), a.scales.repeat(1, M), K)
    y = B.matmul(rows, w, out_dtype=torch.bfloat16).double()[0]
    assert ((y - exact).abs() <= 2.0 ** -12 * mag + 2.0 ** -8 * exact.abs()).all()
