"""How exact the norm's statistics are: sums over a row are pairwise, rstd is the
correctly rounded one but for a hundredth of an ulp."""
import numpy as np
import pytest
import torch

from neuroflow_amd import norm as L
from neuroflow_amd import workloads as WL

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("D", [128, 1024, 4096])
def test_rstd(gpu, D):
    """Rows of +a and -a, a of eight bits: mean 0, variance a^2, every sum on
    the way exact, so that variance + eps is rounded once and known."""
    rng = np.random.default_rng(D)
    a = (rng.integers(128, 256, 2048) * np.exp2(rng.integers(-14, 8, 2048))).astype(np.float32)
    x = torch.from_numpy(a[:, None] * np.where(np.arange(D) % 2, -1, 1).astype(np.float32)).cuda()
    for eps in [0.0, 1e-5, *np.exp2(rng.uniform(-12, 12, 10))]:
        eps = np.float32(eps)
        _, mean, rstd = L.layer_norm(x, eps=float(eps), return_stats=True)
        v = (a.astype(np.float64) ** 2 + np.float64(eps)).astype(np.float32)
        want = 1 / np.sqrt(v.astype(np.float64))
        ulp = np.spacing(want.astype(np.float32)).astype(np.float64)
        assert not mean.any()
        assert (np.abs(rstd.cpu().numpy() - want) <= 0.51 * ulp).all()


@pytest.mark.parametrize("D", [256, 1024, 4096])
def test_mean(gpu, D):
    """Normal values: an addition's rounding is 0.42 U of its result in the rms (a
    uniform error of half an ulp, mantissas by their logarithm), and a pairwise
    sum of D has log2 D levels of them, each of the whole sum's variance; one
    more for the waves' sums, which are joined in turn, and 8% for the draw."""
    x = WL.normal(700 + D, (32768, D)).astype(np.float32)
    _, mean, _ = L.layer_norm(torch.from_numpy(x).cuda(), return_stats=True)
    want = x.astype(np.float64).mean(axis=1)
    err = np.linalg.norm(mean.double().cpu().numpy() - want) / np.linalg.norm(want)
    levels = np.log2(D) + (D > 2048)
    assert err <= 1.08 * 0.4247 * U * np.sqrt(levels), err
