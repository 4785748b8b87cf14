"""Clipping at the ends of max_norm's range."""
import math

import pytest
import torch

from neuroflow_amd import grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [0.0, 1.0, 3e38, float("inf")])
def test_no_bound(gpu, value):
    """An infinite bound clips nothing, in place or not, whatever the norm."""
    ts = [torch.linspace(-1, 1, 1000, device="cuda"), torch.ones(20, device="cuda", dtype=torch.bfloat16)]
    ts[0][3] = value
    before, outs = [t.clone() for t in ts], [torch.zeros_like(t) for t in ts]
    n = grads.clip_by_global_norm(ts, math.inf, out=outs)
    assert all(torch.equal(a, b) for a, b in zip(outs, before))
    assert torch.equal(grads.clip_by_global_norm(ts, math.inf), n) and all(torch.equal(a, b) for a, b in zip(ts, before))
    assert bool(torch.isinf(n)) == (value == math.inf)


def test_no_bound_and_a_nan(gpu):
    ts = [torch.ones(100, device="cuda"), torch.ones(20, device="cuda", dtype=torch.bfloat16)]
    ts[1][0] = float("nan")
    assert bool(torch.isnan(grads.clip_by_global_norm(ts, math.inf))) and all(bool(t.isnan().all()) for t in ts)
