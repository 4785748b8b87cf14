"""examples/norm_fp8_layer.py: training lowers the loss, and the trained layer
serves single tokens as it serves a batch."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "norm_fp8_layer.py"


def _example():
    spec = importlib.util.spec_from_file_location("norm_fp8_layer", EXAMPLE)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_and_serving(gpu, dtype):
    m = _example()
    losses, layer = m.train(steps=40, tokens=1000, d_in=200, d_out=136, dtype=dtype)
    # Plain gradient descent on a noiseless linear teacher: the loss falls by far more than this.
    assert losses[-1] < 0.1 * losses[0]
    served = m.ServedProjection(layer)
    x = torch.randn(5, 200, device="cuda").to(dtype)
    batch = served(x)
    y, _ = layer.forward(x)
    for i in range(5):
        one = served(x[i:i + 1])
        if dtype == torch.float32:
            # The same codes; products and block sums differ in order alone.
            assert torch.allclose(one[0], batch[i], rtol=0, atol=1e-4 * float(batch.abs().max()))
        assert one.shape == (1, 136) and one.dtype == dtype
    if dtype == torch.float32:
        assert torch.allclose(batch, y, rtol=0, atol=1e-4 * float(y.abs().max()))
