"""Block-FP8 products whose exact results are known, at a size for every tile
and split (tests/block_cuts.py).

Codes of -3 .. 3 under scales of 1/2, 1 and 2: a block's 128 products add up to
at most 1152 and a result to at most 36 K < 2^20 quarters, so every sum is exact
in fp32 whatever its order, the FP8 instruction's too (its terms lie within four
bits of each other), and the result has to be the exact one, rounded once.  A
product lost, doubled or under another block's scale shows in any type."""
import pytest
import torch

from block_cuts import BF16, CUTS, F32
from neuroflow_amd import block_fp8 as B
from test_block_cuts import cut

pytestmark = pytest.mark.gpu

TYPES = {F32: torch.float32, BF16: torch.bfloat16}
CODES = [0x00, 0x38, 0x40, 0x44, 0xB8, 0xC0, 0xC4]      # 0, 1, 2, 3, -1, -2, -3


def _operand(g, rows, K, weight):
    """(BlockFp8, its values in float64) of small whole numbers."""
    kb = -(-K // 128)
    codes = torch.tensor(CODES, dtype=torch.uint8, device="cuda")[
        torch.randint(len(CODES), (rows, kb * 128), generator=g, device="cuda")]
    codes[:, K:] = 0
    n = -(-rows // 128) if weight else rows
    scales = torch.exp2(torch.randint(-1, 2, (kb, n), generator=g, device="cuda").float())
    v = codes.view(torch.float8_e4m3fn).float().double().view(rows, kb, 128)
    s = scales.double().t()
    if weight:
        s = s.repeat_interleave(128, 0)[:rows]
    return B.BlockFp8(codes, scales, K), (v * s[:, :, None]).view(rows, -1)


@pytest.mark.parametrize("M,N,K,out,edge,splits", CUTS)
def test_exact(gpu, M, N, K, out, edge, splits):
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert cut(M, N, K, out) == (edge, splits)
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a, av = _operand(g, M, K, False)
    bias = torch.randint(-9, 10, (N,), generator=g, device="cuda").float()
    for weight in (True, False):
        w, wv = _operand(g, N, K, weight)
        want = av @ wv.t()
        y = B.matmul(a, w, out_dtype=TYPES[out])
        assert torch.equal(y, want.float().to(TYPES[out])), (y.double() - want).abs().max()
        y = B.matmul(a, w, bias, "relu", TYPES[out])
        assert torch.equal(y, (want + bias).clamp(min=0).float().to(TYPES[out]))


@pytest.mark.parametrize("M,N,K,dtype", [(3900, 600, 4090, BF16), (65500, 600, 250, BF16), (5003, 1544, 1000, F32),
                                         (700, 9000, 500, BF16), (40, 130, 2049, BF16), (40, 130, 2049, F32)])
def test_backward_is_the_products_of_the_codes(gpu, M, N, K, dtype):
    """dx and dW are, bit for bit, matmul's results on dy's codes: the kernels
    that test_exact holds to the exact ones (dx of the first two in 256 x 256 tiles)."""
    if M > 1000 and dtype == BF16 and torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert cut(M, K, N, dtype)[0] == 256
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    dy = torch.randn(M, N, generator=g, device="cuda").to(TYPES[dtype])
    xc = B.quantise_columns(torch.randn(M, K, generator=g, device="cuda"))
    _, wt = B.quantise_weight(torch.randn(N, K, generator=g, device="cuda"), transposed=True)
    dx, dw, _ = B.linear_backward(dy, xc, wt)
    rows, cols = B.quantise_both(dy)
    assert torch.equal(dx, B.matmul(rows, wt, out_dtype=TYPES[dtype]))
    assert torch.equal(dw, B.matmul(cols, xc))
