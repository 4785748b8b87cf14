"""The norm kernels' loops over rows: more rows than all workgroups hold at
once, at a width for every form of the kernels, against the formulas in 64 bits.

A workgroup of the forward kernels holds at most 16 rows, and at most eight of 256
threads (two of 1024) run on a CU; the backward pass has a workgroup a CU, of at
most 64 rows.  Every row has a level and a mean of its own, so that statistics
of another row, or a sum of another round, show."""
import numpy as np
import pytest
import torch

import block_reference as R
from neuroflow_amd import block_fp8 as B
from neuroflow_amd import norm as L

pytestmark = pytest.mark.gpu

CUS = 256
F32, BF16 = torch.float32, torch.bfloat16


def _data(seed, M, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, D, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(M, 1, generator=g, device="cuda"))
    x += 3 * torch.randn(M, 1, generator=g, device="cuda")
    w = 1 + 0.3 * torch.randn(D, generator=g, device="cuda")
    b = 0.3 * torch.randn(D, generator=g, device="cuda")
    dy = torch.randn(M, D, generator=g, device="cuda").to(dtype)
    return x.to(dtype), w, b, dy


def _np(t):
    return t.double().cpu().numpy()


def _near(got, want, tol, what):
    over = np.abs(_np(got) - want) - tol
    assert np.isfinite(over).all() and (over <= 0).all(), f"{what}: {over.max():.3g} over its bound at {np.unravel_index(over.argmax(), over.shape)}"


# Width, rows of the forward pass: twice the most that run at once, and a remainder.
FORWARD = [(100, 16), (200, 16), (256, 16), (400, 4), (1001, 4), (2000, 4), (4096, 1), (8000, 1), (12000, 1 / 4), (17000, 1 / 2)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,rows", FORWARD)
def test_forward(gpu, D, rows, dtype):
    M = int(2 * 8 * CUS * rows) + 5
    x, w, b, _ = _data(800 + D, M, D, dtype)
    y, mean, rstd = L.layer_norm(x, w, b, 1e-5, return_stats=True)
    q, mq, rq = L.layer_norm_fp8(x, w, b, 1e-5, return_stats=True)
    assert torch.equal(mean, mq) and torch.equal(rstd, rq)
    # All rows in turns of at most four million values.
    step = max(1, (1 << 22) // D)
    for r in range(0, M, step):
        xd = _np(x[r:r + step])
        want, m64, r64 = R.norm(xd, _np(w), _np(b), 1e-5)
        ty, tm, tr = R.norm_tols(xd, _np(w), _np(b), 1e-5, want, r64, dtype == BF16)
        _near(mean[r:r + step], m64, tm, "mean")
        _near(rstd[r:r + step], r64, tr, "rstd")
        _near(y[r:r + step], want, ty, "y")
    # The codes are those of the fp32 result, whatever the input's type.
    full = B.quantise(L.layer_norm(x.float(), w, b, 1e-5))
    assert torch.equal(q.scales, full.scales) and torch.equal(q.codes, full.codes)


# Width, rows of a workgroup (fp32, bf16).
BACKWARD = [(96, 64, 64), (200, 64, 64), (400, 16, 16), (1001, 16, 16), (2000, 4, 4), (4096, 2, 4), (8000, 1, 1), (12000, 1, 1),
            (17000, 1, 1)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,g32,g16", BACKWARD)
def test_backward(gpu, D, g32, g16, dtype):
    M = 2 * CUS * (g32 if dtype == F32 else g16) + 3
    x, w, _, dy = _data(900 + D, M, D, dtype)
    xd, dyd = _np(x), _np(dy)
    m32 = x.double().mean(1).float()
    r32 = (x.double().var(1, unbiased=False) + 1e-5).rsqrt().float()
    dx, dw, db = L.layer_norm_backward(dy, x, w, m32, r32)
    want, dw64, db64, h, g = R.norm_grad(dyd, xd, _np(w), _np(m32), _np(r32))
    t, tw, tb = R.norm_grad_tols(dyd, xd, h, g, _np(r32), want, dtype == BF16)
    _near(dx, want, t, "dx")
    _near(dw, dw64, tw, "dweight")
    _near(db, db64, tb, "dbias")
    # A row's part in the sums: take away one row of the last round and one of the first.
    for r in (0, M - 1):
        dy2 = dy.clone()
        dy2[r] = 0
        _, dw2, db2 = L.layer_norm_backward(dy2, x, w, m32, r32)
        _near(dw - dw2, dyd[r] * h[r], 2 * tw, "dweight's part of a row")
        _near(db - db2, dyd[r], 2 * tb, "dbias's part of a row")
