"""norm and block_fp8 next to autograd: results carry no graph, and a tensor
written through `out` counts as changed."""
import pytest
import torch

from neuroflow_amd import block_fp8 as B
from neuroflow_amd import norm as L

pytestmark = pytest.mark.gpu


def test_out_raises_the_version(gpu):
    x = torch.randn(8, 64, device="cuda")
    v = x._version
    L.layer_norm(x)
    assert x._version == v
    L.layer_norm(x, out=x)
    assert x._version == v + 1
    out = torch.empty(20, 64, device="cuda")
    v = out._version
    L.layer_norm(x, out=out[4:12])          # a view shares its tensor's version
    assert out._version == v + 1


def test_a_graph_that_saved_x_notices(gpu):
    x, p = torch.randn(8, 64, device="cuda"), torch.randn(8, 64, device="cuda", requires_grad=True)
    y = (x * p).sum()
    L.layer_norm(x, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors(gpu):
    with torch.inference_mode():
        x = torch.randn(8, 64, device="cuda")
        want = L.layer_norm(x)
        assert torch.equal(L.layer_norm(x, out=x), want)
    y = x.clone()
    L.layer_norm(y, out=x)                  # written outside of the mode, as plain memory
    assert torch.equal(x, L.layer_norm(y))


def test_no_graph(gpu):
    x = torch.randn(8, 256, device="cuda", requires_grad=True)
    w = B.quantise_weight(torch.randn(128, 256, device="cuda", requires_grad=True))
    for t in (L.layer_norm(x), B.linear(x, w), B.quantise(x).scales):
        assert not t.requires_grad
    with pytest.raises(ValueError, match="requires grad"):
        L.layer_norm(x, out=x)
    with torch.no_grad():
        L.layer_norm(x, out=x)
