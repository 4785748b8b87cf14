"""RMS norm into block FP8: the codes past the last column are zero in every row,
also where the row's 1 / rms is a NaN or an infinity."""
import pytest
import torch

from neuroflow_amd import norm as L
from residual_reference import DTYPES, gen, rows

pytestmark = pytest.mark.gpu
# Widths short of a whole block, of every register kernel and of the one past them.
WIDTHS = [1, 7, 100, 130, 250, 300, 600, 1001, 1100, 2100, 4097, 5000, 8200, 12001, 16300, 17001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("weighted", [False, True])
def test_padding(gpu, D, dtype, weighted):
    g = gen(D)
    x, r = rows(7, D, dtype, g), rows(7, D, dtype, g)
    w = 1 + 0.1 * torch.randn(D, generator=g, device="cuda") if weighted else None
    x[1, D // 2] = float("nan")
    x[2, D - 1], r[2, D - 1] = float("inf"), float("-inf")
    x[3, 0] = float("inf")
    x[4], r[4] = 0, 0
    for eps in (0.0, 1e-5):
        for residual in (None, r):
            q = L.rms_norm_fp8(x, w, eps, residual=residual)
            q = q[0] if residual is not None else q
            assert q.codes.shape[1] > D and not bool(q.codes[:, D:].any()), (eps, residual is None)
            y = L.rms_norm(x, w, eps, residual=residual)
            y = y[0] if residual is not None else y
            # What is a NaN stays one: the byte 0x7F, and no other.
            bad = torch.isnan(y)
            assert bool(bad[1].all()) and torch.equal(q.codes[:, :D] == 0x7F, bad)
