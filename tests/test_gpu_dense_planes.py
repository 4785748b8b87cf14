"""fp32 products whose operands both need more than their first bf16 part: known
exactly, through every kernel and cut; at the values that the parts left out
weigh most in; and in the 2-norm against 64 bits."""
import pytest
import torch

from neuroflow_amd import dense
from residual_reference import gen, rows
from test_gpu_dense import CUTS

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
# The few-row kernel of one and of two row groups, pieces of K that end anywhere.
FEW = [(1, 1, 1), (1, 64, 40), (3, 33, 100), (16, 300, 130), (17, 1000, 4096), (32, 257, 300), (1, 4096, 4096), (20, 4100, 1000)]


def whole(m, n, g, keep):
    """Whole numbers of ten bits, h and m of both parts not zero, at most `keep` not 0 in a row."""
    v = torch.randint(513, 1024, (m, n), generator=g, device="cuda").float()
    v = v * (2 * torch.randint(0, 2, (m, n), generator=g, device="cuda") - 1)
    if n > keep:
        v[:, torch.randperm(n, generator=g, device="cuda")[keep:]] = 0
    return v


def check_exact(M, K, N):
    """Products are below 2^20, and sums of sixteen below 2^24."""
    g = gen(M + K + N)
    x, W = whole(M, K, g, 16), whole(N, K, g, K)
    assert torch.equal(dense.linear(x, W), (x.double() @ W.double().t()).float())
    dy = whole(M, N, g, 16)
    dy[torch.randperm(M, generator=g, device="cuda")[16:]] = 0
    x = whole(M, K, g, K)
    dx, dW, db, _ = dense.linear_backward(dy, x, W)
    assert torch.equal(dx, (dy.double() @ W.double()).float())
    assert torch.equal(dW, (dy.double().t() @ x.double()).float())
    assert torch.equal(db, dy.double().sum(0).float())


@pytest.mark.parametrize("M,K,N", FEW)
def test_exact_few(gpu, M, K, N):
    check_exact(M, K, N)


@pytest.mark.parametrize("M,K,N", CUTS)
def test_exact_cuts(gpu, M, K, N):
    check_exact(M, K, N)


# 1 + 2^-8 - 2^-16 + 2^-17 - 2^-23 and its neighbours: the middle part is near 2^-8 of the
# value and the last near 2^-17, the most that each can be.
WORST = [1 + 2.0 ** -8 - 2.0 ** -16 + 2.0 ** -17 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -7 + 2.0 ** -8 - 2.0 ** -16 + 2.0 ** -17,
         1 - 2.0 ** -9 + 2.0 ** -17 - 2.0 ** -24, 1 + 2.0 ** -23, 2 - 2.0 ** -23]


@pytest.mark.parametrize("M", [1, 20, 33, 200, 1025])
def test_parts_left_out(gpu, M):
    """One product a result: off by what the three least parts come to, 2^-24 of it
    (|m| <= 2^-8 and |l| <= 2^-17 of a value's power of two), and by the sums of the
    six that are formed, each within a step of fp32."""
    v = torch.tensor(WORST, device="cuda")
    v = torch.cat([v, -v, v * 2.0 ** 40, v * 2.0 ** -40])
    x = v[torch.arange(M, device="cuda") % len(v)][:, None].contiguous()
    W = v[:, None].contiguous()
    want = x.double() @ W.double().t()
    off = (dense.linear(x, W).double() - want).abs() / want.abs()
    assert float(off.max()) <= (1 + 6 * 2) * U


def far(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("M,K,N", [(1, 64, 300), (20, 33, 500), (32, 64, 64), (64, 64, 64), (40, 20, 64), (64, 50, 33)])
def test_two_norm(gpu, M, K, N):
    """Sums of at most 64 terms take at most two additions of each of the six products
    to a result, each off by at most a step of fp32 (2 U) of a sum whose 2-norm over all
    results is at most the last one's; the parts left out are 2^-24 of the terms and
    the last rounding is half a step.  That is 1.6e-6; without the product of the middle parts
    the results are off by 2.5e-6."""
    g = gen(M + K)
    x, W, dy = rows(M, K, torch.float32, g), torch.randn(N, K, generator=g, device="cuda"), rows(M, N, torch.float32, g)
    most = lambda k: (2 * 6 * -(-k // 32) + 2) * U
    assert far(dense.linear(x, W), x.double() @ W.double().t()) <= most(K)
    if max(M, N) <= 64:
        dx, dW, _, _ = dense.linear_backward(dy, x, W)
        assert far(dx, dy.double() @ W.double()) <= most(N)
        assert far(dW, dy.double().t() @ x.double()) <= most(M)
