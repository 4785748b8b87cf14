"""Layer norm forward, into block FP8, and backward, against the formulas in
64 bits (tests/block_reference.py; its bounds are derived there)."""
import numpy as np
import pytest
import torch

import block_reference as R
from neuroflow_amd import _lib
from neuroflow_amd import block_fp8 as B
from neuroflow_amd import norm as L
from neuroflow_amd import workloads as WL

pytestmark = pytest.mark.gpu

# One to a few lanes, around a wave's vectors, a block, the register kernels' widths and past them.
WIDTHS = [1, 3, 7, 64, 100, 127, 128, 129, 256, 1000, 1001, 1024, 1025, 2047, 4096, 4100, 5000, 16384, 16391, 40000]


def _data(seed, M, D, dtype, level=3.0):
    x = (WL.normal(seed, (M, D)) * np.exp(0.5 * WL.normal(seed + 1, (M, 1))) + level).astype(np.float32)
    t = torch.from_numpy(x).cuda().to(dtype)
    w, b = 1 + 0.3 * WL.normal(seed + 2, (D,)), 0.3 * WL.normal(seed + 3, (D,))
    return t, t.double().cpu().numpy(), w.astype(np.float32), b.astype(np.float32)


def _cuda(a):
    return None if a is None else torch.from_numpy(a).cuda()


def _near(got, want, tol, what):
    got = got.double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    over = np.abs(got - want) - tol
    assert np.isfinite(got).all() and (over <= 0).all(), f"{what}: {over.max():.3g} over its bound at {np.unravel_index(over.argmax(), over.shape)}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", WIDTHS)
def test_forward(gpu, D, dtype):
    M = 5 if D > 2048 else 37
    x, xd, w, b = _data(10 + D, M, D, dtype)
    for ww, bb in ((w, b), (None, None), (w, None), (None, b)):
        y, mean, rstd = L.layer_norm(x, _cuda(ww), _cuda(bb), 1e-5, return_stats=True)
        want, m64, r64 = R.norm(xd, ww, bb, 1e-5)
        ty, tm, tr = R.norm_tols(xd, ww, bb, 1e-5, want, r64, dtype == torch.bfloat16)
        _near(mean, m64, tm, "mean")
        _near(rstd, r64, tr, "rstd")
        _near(y, want, ty, "y")
        assert torch.equal(L.layer_norm(x, _cuda(ww), _cuda(bb), 1e-5), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 63, 255, 1030, 9001])
def test_forward_row_counts(gpu, M, dtype):
    x, xd, w, b = _data(50 + M, M, 200, dtype)
    y = L.layer_norm(x, _cuda(w), _cuda(b))
    want, _, r64 = R.norm(xd, w, b, 1e-5)
    _near(y, want, R.norm_tols(xd, w, b, 1e-5, want, r64, dtype == torch.bfloat16)[0], "y")


def test_forward_constant_and_offset_rows(gpu):
    """A constant row gives the bias (variance 0, eps alone); a row far from
    zero keeps its deviations (no sum of squares about zero)."""
    x = np.full((3, 300), 7.25, np.float32)
    x[1] = 4096.0 + WL.normal(61, (300,)).astype(np.float32)
    x[2] = 0.0
    b = WL.normal(62, (300,)).astype(np.float32)
    y, mean, rstd = L.layer_norm(_cuda(x), None, _cuda(b), 1e-5, return_stats=True)
    assert torch.equal(y[0], _cuda(b)) and torch.equal(y[2], _cuda(b)) and float(mean[0]) == 7.25
    want, _, r64 = R.norm(x.astype(np.float64), None, b, 1e-5)
    _near(y, want, R.norm_tols(x.astype(np.float64), None, b, 1e-5, want, r64, False)[0], "y")


def test_forward_nonfinite_stays_in_its_row(gpu):
    x, _, w, b = _data(70, 6, 515, torch.float32)
    clean = L.layer_norm(x, _cuda(w), _cuda(b))
    x2 = x.clone()
    x2[2, 100], x2[4, 514] = float("nan"), float("inf")
    y = L.layer_norm(x2, _cuda(w), _cuda(b))
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all()
    keep = [0, 1, 3, 5]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 130, 1001, 4098, 17000])
def test_strides_in_place_and_streams(gpu, D, dtype):
    """Rows at any stride and element offset; out over x; a stream of its own."""
    M = 21
    x, xd, w, b = _data(80 + D, M, D, dtype)
    plain = L.layer_norm(x, _cuda(w), _cuda(b))
    wide = torch.full((M, D + 5), 9.0, dtype=dtype, device="cuda")
    wide[:, 1:1 + D] = x
    out = torch.full((M, D + 3), 5.0, dtype=dtype, device="cuda")
    L.layer_norm(wide[:, 1:1 + D], _cuda(w), _cuda(b), out=out[:, 2:2 + D])
    assert torch.equal(out[:, 2:2 + D], plain)
    assert (out[:, :2] == 5).all() and (out[:, 2 + D:] == 5).all()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        z = x.clone()
        L.layer_norm(z, _cuda(w), _cuda(b), out=z)
    st.synchronize()
    assert torch.equal(z, plain)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", WIDTHS)
def test_fp8(gpu, D, dtype):
    """Codes and scales are those of the quantise applied to some y within the
    norm's bound: each scale is within that of the 64-bit y's, and each code
    times its scale within half a code step of y."""
    M = 5 if D > 2048 else 37
    x, xd, w, b = _data(90 + D, M, D, dtype)
    q, mean, rstd = L.layer_norm_fp8(x, _cuda(w), _cuda(b), 1e-5, return_stats=True)
    want, m64, r64 = R.norm(xd, w, b, 1e-5)
    ty, tm, tr = R.norm_tols(xd, w, b, 1e-5, want, r64, False)
    _near(mean, m64, tm, "mean")
    _near(rstd, r64, tr, "rstd")
    kb = R.blocks(D)
    pad = np.zeros((M, kb * 128))
    pad[:, :D] = want
    tpad = np.zeros((M, kb * 128))
    tpad[:, :D] = ty
    amax = np.abs(pad.reshape(M, kb, 128)).max(axis=2)
    tmax = tpad.reshape(M, kb, 128).max(axis=2)
    s = q.scales.double().cpu().numpy().T
    assert (np.abs(s * 448 - amax) <= tmax + 4 * R.U * amax).all()
    codes = q.codes.cpu().numpy()
    assert (codes[:, D:] == 0).all()
    v = R.values(codes, q.scales.cpu().numpy())
    full = np.repeat(s, 128, axis=1)
    # Half a step: 2^-4 of a normal value (4 significant bits), 2^-10 of the scale below 2^-6,
    # and the codec's cap there (up to a whole step, 2^-9).
    step = np.maximum(np.abs(pad) * 2.0 ** -4, full * 2.0 ** -9)
    assert (np.abs(v - pad) <= step * (1 + 1e-5) + tpad).all()


@pytest.mark.parametrize("D", [256, 1000, 4096, 20000])
def test_fp8_is_the_quantise_of_the_fp32_norm(gpu, D):
    """For fp32 rows, layer_norm_fp8 gives the bits of quantise(layer_norm)."""
    x, _, w, b = _data(95 + D, 19, D, torch.float32)
    a = L.layer_norm_fp8(x, _cuda(w), _cuda(b))
    c = B.quantise(L.layer_norm(x, _cuda(w), _cuda(b)))
    assert torch.equal(a.codes, c.codes) and torch.equal(a.scales, c.scales) and a.k == c.k == D


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", WIDTHS)
def test_backward(gpu, D, dtype):
    M = 7 if D > 2048 else 83
    x, xd, w, _ = _data(100 + D, M, D, dtype)
    dy = torch.from_numpy(WL.normal(101 + D, (M, D)).astype(np.float32)).cuda().to(dtype)
    dyd = dy.double().cpu().numpy()
    for ww in (w, None):
        _, m64, r64 = R.norm(xd, None, None, 1e-5)
        mean, rstd = m64.astype(np.float32), r64.astype(np.float32)
        dx, dw, db = L.layer_norm_backward(dy, x, _cuda(ww), _cuda(mean), _cuda(rstd))
        want, ww64, wb64, h, g = R.norm_grad(dyd, xd, ww, mean.astype(np.float64), rstd.astype(np.float64))
        t, tw, tb = R.norm_grad_tols(dyd, xd, h, g, rstd.astype(np.float64), want, dtype == torch.bfloat16)
        _near(dx, want, t, "dx")
        _near(dw, ww64, tw, "dweight")
        _near(db, wb64, tb, "dbias")
        again = L.layer_norm_backward(dy, x, _cuda(ww), _cuda(mean), _cuda(rstd))
        assert all(torch.equal(p, r) for p, r in zip((dx, dw, db), again))


@pytest.mark.parametrize("M", [1, 2, 5, 255, 256, 257, 1031, 20011])
def test_backward_row_counts(gpu, M):
    D = 96
    x, xd, w, _ = _data(110 + M, M, D, torch.float32)
    dy = torch.from_numpy(WL.normal(111 + M, (M, D)).astype(np.float32)).cuda()
    dyd = dy.double().cpu().numpy()
    _, m64, r64 = R.norm(xd, None, None, 1e-5)
    mean, rstd = m64.astype(np.float32), r64.astype(np.float32)
    dx, dw, db = L.layer_norm_backward(dy, x, _cuda(w), _cuda(mean), _cuda(rstd))
    want, ww64, wb64, h, g = R.norm_grad(dyd, xd, w, mean.astype(np.float64), rstd.astype(np.float64))
    t, tw, tb = R.norm_grad_tols(dyd, xd, h, g, rstd.astype(np.float64), want, False)
    _near(dx, want, t, "dx")
    _near(dw, ww64, tw, "dweight")
    _near(db, wb64, tb, "dbias")


def test_backward_against_differences(gpu):
    """<dx, v>, <dweight, u>, <dbias, u> against central differences of the
    64-bit forward: third-order remainder 1e-8 of the step's, fp32 gradients."""
    M, D, hstep = 6, 77, 1e-4
    x, xd, w, b = _data(120, M, D, torch.float32, level=0.5)
    dyd = WL.normal(121, (M, D)).astype(np.float32).astype(np.float64)
    _, mean, rstd = L.layer_norm(x, _cuda(w), _cuda(b), 1e-5, return_stats=True)
    dx, dw, db = L.layer_norm_backward(torch.from_numpy(dyd.astype(np.float32)).cuda(), x, _cuda(w), mean, rstd)
    v, u = WL.normal(122, (M, D)).astype(np.float64), WL.normal(123, (D,)).astype(np.float64)
    w64, b64 = w.astype(np.float64), b.astype(np.float64)

    def f(xx, ww, bb):
        return (dyd * R.norm(xx, ww, bb, 1e-5)[0]).sum()

    def diff(g):
        return (g(hstep) - g(-hstep)) / (2 * hstep)

    scale = np.abs(dyd).sum()
    for got, want in (((dx.double().cpu().numpy() * v).sum(), diff(lambda e: f(xd + e * v, w64, b64))),
                      ((dw.double().cpu().numpy() * u).sum(), diff(lambda e: f(xd, w64 + e * u, b64))),
                      ((db.double().cpu().numpy() * u).sum(), diff(lambda e: f(xd, w64, b64 + e * u)))):
        assert abs(got - want) <= 2e-5 * scale


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 130, 1001, 4098, 17000])
def test_backward_strides_and_in_place(gpu, D, dtype):
    """Strided dy and x through the wrapper; dx over dy, and over x, through the C entry."""
    M = 19
    x, xd, w, _ = _data(130 + D, M, D, dtype)
    dy = torch.from_numpy(WL.normal(131 + D, (M, D)).astype(np.float32)).cuda().to(dtype)
    _, mean, rstd = L.layer_norm(x, return_stats=True)
    dx, dw, db = L.layer_norm_backward(dy, x, _cuda(w), mean, rstd)
    xs = torch.zeros(M, D + 3, dtype=dtype, device="cuda")
    ys = torch.zeros(M, 2 * D + 1, dtype=dtype, device="cuda")
    xs[:, 1:1 + D], ys[:, D:2 * D] = x, dy
    got = L.layer_norm_backward(ys[:, D:2 * D], xs[:, 1:1 + D], _cuda(w), mean, rstd)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dw) and torch.equal(got[2], db)
    lib, wt = _lib.lib(), _cuda(w)
    n = _lib.C.c_size_t()
    assert lib.nflow_layer_norm_backward_workspace(M, D, _lib.C.byref(n)) == 0
    ws = torch.empty(max(n.value, 1), dtype=torch.uint8, device="cuda")
    for over_x in (False, True):
        p, q = dy.clone(), x.clone()
        out = q if over_x else p
        rc = lib.nflow_layer_norm_backward(p.data_ptr(), q.data_ptr(), B._DTYPES[x.dtype], M, D, D, D, wt.data_ptr(),
                                           mean.data_ptr(), rstd.data_ptr(), out.data_ptr(), D, None, None,
                                           ws.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(out, dx)


def test_empty(gpu):
    x = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    y, mean, rstd = L.layer_norm(x, w, w, return_stats=True)
    assert y.shape == (0, 64) and mean.numel() == 0
    assert L.layer_norm_fp8(x, w, w).codes.shape == (0, 128)
    dx, dw, db = L.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_refusals(gpu):
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    with pytest.raises(TypeError):
        L.layer_norm(x.half())
    with pytest.raises(TypeError):
        L.layer_norm(x.cpu())
    with pytest.raises(TypeError):
        L.layer_norm(x, w.bfloat16())
    with pytest.raises(ValueError):
        L.layer_norm(x, w[:63])
    with pytest.raises(ValueError):
        L.layer_norm(x.t())
    with pytest.raises(ValueError):
        L.layer_norm(x, out=torch.zeros(4, 63, device="cuda"))
    with pytest.raises(_lib.NflowError):
        L.layer_norm(x, eps=-1.0)
    with pytest.raises(_lib.NflowError):
        L.layer_norm(x, eps=float("nan"))
    with pytest.raises(_lib.NflowError):
        L.layer_norm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(ValueError):
        L.layer_norm_backward(x[:3], x, w, torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        L.layer_norm_backward(x, x, w, torch.zeros(3, device="cuda"), torch.zeros(4, device="cuda"))
    with pytest.raises(TypeError):
        L.layer_norm_backward(x, x, w, None, torch.zeros(4, device="cuda"))


def test_graph_replays(gpu):
    """Captured once, replayed on new inputs with eager calls between."""
    x, _, w, b = _data(140, 300, 1000, torch.bfloat16)
    w, b, dy = _cuda(w), _cuda(b), torch.randn(300, 1000, device="cuda").bfloat16()

    def step():
        y, mean, rstd = L.layer_norm(x, w, b, return_stats=True)
        q = L.layer_norm_fp8(x, w, b)
        return (y, q.codes, q.scales, *L.layer_norm_backward(dy, x, w, mean, rstd))

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(3):
        x.copy_(_data(141 + k, 300, 1000, torch.bfloat16)[0])
        want = [t.clone() for t in step()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, r) for p, r in zip(out, want))


def test_rows_past_32_bit_offsets(gpu):
    """More than 2^32 elements: the last rows are as those of a small call."""
    D = 4096
    M = (1 << 20) + 3
    x = torch.zeros(M, D, dtype=torch.bfloat16, device="cuda")
    tail, _, w, b = _data(150, 5, D, torch.bfloat16)
    x[-5:] = tail
    w, b = _cuda(w), _cuda(b)
    y, mean, rstd = L.layer_norm(x, w, b, return_stats=True)
    small, m5, r5 = L.layer_norm(tail, w, b, return_stats=True)
    assert torch.equal(y[-5:], small) and torch.equal(mean[-5:], m5) and torch.equal(rstd[-5:], r5)
    del y
    q, q5 = L.layer_norm_fp8(x, w, b), L.layer_norm_fp8(tail, w, b)
    assert torch.equal(q.codes[-5:], q5.codes) and torch.equal(q.scales[:, -5:], q5.scales)
    del q
    dx, _, _ = L.layer_norm_backward(x, x, w, mean, rstd)
    assert torch.equal(dx[-5:], L.layer_norm_backward(tail, tail, w, m5, r5)[0])
