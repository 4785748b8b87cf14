"""Results that share memory with an input in another way than row for row are
refused: the rows of different workgroups would read what others have written."""
import pytest
import torch

from neuroflow_amd import _lib
from neuroflow_amd import norm as L

P = 1 << 20        # a non-null, aligned address; never followed: every call that gets it is refused


def forward(y, ldy, M=8, D=64, ldx=64, dtype=0):
    return _lib.lib().nflow_layer_norm_forward(P, dtype, M, D, ldx, None, None, 1e-5, y, ldy, None, None, None)


@pytest.mark.parametrize("dtype", [0, 1])
def test_forward_is_refused(dtype):
    e = 2 if dtype else 4
    for y, ldy in ((P + 64 * e, 64), (P - 64 * e, 64), (P + e, 64), (P - 7 * 64 * e, 64), (P, 65), (P + 32 * e, 200)):
        assert forward(y, ldy, dtype=dtype) == _lib.INVALID_ARG, (y - P, ldy)
        assert b"layer_norm_forward" in _lib.lib().nflow_last_error()
    assert forward(P + 4, 64, M=1) == _lib.INVALID_ARG
    for off in (40, 100, -40):                                # rows of 64 in strides of 128: these meet
        assert forward(P + off * e, 128, ldx=128, dtype=dtype) == _lib.INVALID_ARG


@pytest.mark.parametrize("over", ["dy", "x"])
def test_backward_is_refused(over):
    far, ws = P + (1 << 24), P + (1 << 25)
    dy, x = (P, far) if over == "dy" else (far, P)
    for dx, lddx in ((P + 256, 64), (P, 72), (P - 256, 64)):
        assert _lib.lib().nflow_layer_norm_backward(dy, x, 0, 8, 64, 64, 64, None, P + (1 << 26), P + (1 << 26), dx, lddx,
                                                    None, None, ws, 1 << 20, None) == _lib.INVALID_ARG
        assert b"layer_norm_backward" in _lib.lib().nflow_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_side_by_side_and_in_place(gpu, dtype):
    """Disjoint rows of one tensor, and the same rows, are taken."""
    buf = torch.randn(300, 200, device="cuda").to(dtype)
    x = buf[:, :96]
    want = L.layer_norm(x.contiguous())
    keep = buf[:, 196:].clone()
    assert torch.equal(L.layer_norm(x, out=buf[:, 100:196]), want) and torch.equal(buf[:, 196:], keep)
    assert torch.equal(L.layer_norm(x, out=x), want) and torch.equal(x, want)
    with pytest.raises(_lib.NflowError):
        L.layer_norm(buf[:-1, :96], out=buf[1:, :96])
    with pytest.raises(_lib.NflowError):
        L.layer_norm(buf[:, :96], out=buf[:, 50:146])
