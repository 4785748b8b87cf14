"""RMS norm with the residual's addition against its formula in 64 bits:
forward, into block FP8, backward; widths of every kernel, odd sizes, strides,
zero rows, infinities, results in place, streams and captured graphs."""
import pytest
import torch

from neuroflow_amd import _lib
from neuroflow_amd import block_fp8 as B
from neuroflow_amd import norm as L
from residual_reference import DTYPES, U, gen, half, rms, rms_chain, rows, within

pytestmark = pytest.mark.gpu
# (rows, columns): one value to rows past the registers' width, and every kernel's widths.
SIZES = [(1, 1), (3, 7), (1, 64), (5, 128), (17, 129), (33, 256), (9, 257), (4, 512), (1, 1000), (300, 1001), (7, 2048),
         (2, 2049), (5, 4096), (3, 4104), (2, 8192), (3, 9000), (2, 16384), (2, 16385), (1, 20001), (2000, 96)]


def inputs(M, D, dtype, seed, stride=None):
    g = gen(seed)
    return (rows(M, D, dtype, g, 2.0, stride), rows(M, D, dtype, g, 1.0, stride and stride + 3),
            1 + 0.3 * torch.randn(D, generator=g, device="cuda"))


def check(x, r, w, eps, y, t, rstd):
    dtype, D = x.dtype, x.shape[-1]
    want, total, rs = rms(x, w, eps, r)
    # Half of the sum's relative error, the root, the product's roundings, t's own.
    rel = (rms_chain(D) / 2 + 8) * U
    within(rstd, rs, rs * rel)
    within(y, want, want.abs() * (rel + half(dtype) * (1 + rel)) + 2.0 ** -133)
    if r is not None:
        within(t, total, total.abs() * (U + half(dtype)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", SIZES)
def test_forward(gpu, M, D, dtype):
    x, r, w = inputs(M, D, dtype, M + D)
    y, t, rstd = L.rms_norm(x, w, 1e-5, residual=r, return_stats=True)
    assert y.dtype == t.dtype == dtype and rstd.dtype == torch.float32 and rstd.shape == (M,)
    check(x, r, w, 1e-5, y, t, rstd)
    y, rstd = L.rms_norm(x, w, 1e-3, return_stats=True)
    check(x, None, w, 1e-3, y, None, rstd)
    assert torch.equal(L.rms_norm(x, None, 1e-3), L.rms_norm(x, torch.ones_like(w), 1e-3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D,stride", [(37, 100, 101), (5, 256, 300), (3, 1025, 1031), (2, 17000, 17001)])
def test_strides(gpu, M, D, dtype, stride):
    """Rows apart, at any element alignment, with NaN between them."""
    x, r, w = inputs(M, D, dtype, 5, stride)
    y, t, rstd = L.rms_norm(x, w, residual=r, return_stats=True)
    check(x, r, w, 1e-5, y, t, rstd)
    same = L.rms_norm(x.contiguous(), w, residual=r.contiguous(), return_stats=True)
    assert all(torch.equal(a, b) for a, b in zip((y, t, rstd), same))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [96, 1000, 17000])
def test_leading_axes_and_no_rows(gpu, dtype, D):
    x, r, w = inputs(24, D, dtype, 6)
    want = L.rms_norm(x, w, residual=r, return_stats=True)
    got = L.rms_norm(x.view(2, 3, 4, D), w, residual=r.view(2, 3, 4, D), return_stats=True)
    assert got[0].shape == got[1].shape == (2, 3, 4, D)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(got, want))
    y, t, rstd = L.rms_norm(x[:0], w, residual=r[:0], return_stats=True)
    assert y.shape == t.shape == (0, D) and rstd.shape == (0,)
    dx, dw = L.rms_norm_backward(x[:0], x[:0], w, rstd)
    assert dx.shape == (0, D) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 500, 4096, 17000])
def test_sum_in_place(gpu, dtype, D):
    """The stream takes the sum: sum_out is the residual, or x, or rows of another stride."""
    x, r, w = inputs(19, D, dtype, 7)
    y, t, rstd = L.rms_norm(x, w, residual=r, return_stats=True)
    for which in (0, 1):
        xs, rs = x.clone(), r.clone()
        to = (xs, rs)[which]
        version = to._version
        y2, t2 = L.rms_norm(xs, w, residual=rs, sum_out=to)
        assert torch.equal(y2, y) and t2 is to and torch.equal(to, t) and to._version == version + 1
        xs, rs = x.clone(), r.clone()
        to = (xs, rs)[which]
        q, t2 = L.rms_norm_fp8(xs, w, residual=rs, sum_out=to)
        assert torch.equal(to, t) and torch.equal(q.codes, L.rms_norm_fp8(x, w, residual=r)[0].codes)
    buf = torch.zeros(19, D + 5, device="cuda", dtype=dtype)
    L.rms_norm(x, w, residual=r, sum_out=buf[:, 2:D + 2])
    assert torch.equal(buf[:, 2:D + 2], t) and not bool(buf[:, :2].any()) and not bool(buf[:, D + 2:].any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", [(1, 1), (5, 128), (17, 129), (40, 256), (9, 1000), (33, 4096), (2, 8200), (3, 16384),
                                 (2, 17001)])
def test_fp8(gpu, M, D, dtype):
    """The codes and scales of rms_norm's fp32 result: of the bf16 or fp32 y they
    are the quantise's wherever that y is the unrounded one."""
    x, r, w = inputs(M, D, dtype, M * D)
    q, t, rstd = L.rms_norm_fp8(x, w, residual=r, return_stats=True)
    y, t2, rstd2 = L.rms_norm(x, w, residual=r, return_stats=True)
    assert torch.equal(t, t2) and torch.equal(rstd, rstd2) and q.k == D
    if dtype == torch.float32:
        want = B.quantise(y)
        assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
    # As values: half a step of e4m3 (2^-4), or of its subnormals' scale.
    full, _, _ = rms(x, w, 1e-5, r)
    scale = q.scales.t().double().repeat_interleave(128, 1)[:, :D]
    got = q.codes.view(torch.float8_e4m3fn).double()[:, :D] * scale
    within(got, full, full.abs() * (2.0 ** -4 + 2.0 ** -18) + scale * 2.0 ** -9)
    assert not bool(q.codes[:, D:].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_rows_and_special_values(gpu, dtype):
    """A row of zeros (1 / sqrt(eps)), of cancelling terms, with infinities and
    NaN; their neighbours are as without them."""
    x, r, w = inputs(8, 300, dtype, 8)
    want = L.rms_norm(x, w, residual=r, return_stats=True)
    x2, r2 = x.clone(), r.clone()
    x2[1], r2[1] = 0, 0
    r2[2] = -x2[2]
    x2[3, 5] = float("inf")
    x2[4, 7] = float("nan")
    x2[5, 9], r2[5, 9] = float("inf"), float("-inf")
    y, t, rstd = L.rms_norm(x2, w, residual=r2, return_stats=True)
    for i in (0, 6, 7):
        assert all(torch.equal(a[i], b[i]) for a, b in zip((y, t, rstd), want))
    for i in (1, 2):
        assert not bool(y[i].any()) and not bool(t[i].any())
        within(rstd[i:i + 1], torch.tensor([1e-5 ** -0.5], device="cuda", dtype=torch.float64), 316.3 * 8 * U)
    assert float(rstd[3]) == 0 and bool(torch.isnan(y[3, 5])) and not bool(y[3, :5].any())
    assert bool(torch.isnan(y[4]).all()) and bool(torch.isnan(y[5]).all()) and bool(torch.isnan(t[5, 9]))
    q, t2 = L.rms_norm_fp8(x2, w, residual=r2)
    ref = L.rms_norm_fp8(x, w, residual=r)[0]
    assert torch.equal(q.codes[[0, 6, 7]], ref.codes[[0, 6, 7]]) and not bool(q.codes[1:3].any())
    y, rstd = L.rms_norm(torch.zeros(2, 40, device="cuda", dtype=dtype), None, 0.0, return_stats=True)
    assert bool(torch.isinf(rstd).all())                       # as the formula has it with eps 0


def reference_backward(dy, x, w, rstd, dsum):
    dy, x, rs = dy.double(), x.double(), rstd.double()[:, None]
    h = x * rs
    g = dy * w.double()
    mean = (g * h).mean(1, keepdim=True)
    dt = rs * (g - h * mean)
    size = rs * (g.abs() + h.abs() * (g * h).abs().mean(1, keepdim=True))
    if dsum is not None:
        dt, size = dt + dsum.double(), size + dsum.double().abs()
    return dt, size, (dy * h).sum(0), (dy * h).abs().sum(0)


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,D", SIZES + [(700, 130), (1500, 300), (600, 2000)])
def test_backward(gpu, M, D, dtype, add):
    x, ds, w = inputs(M, D, dtype, M + 3 * D)
    dy = rows(M, D, dtype, gen(M), 0.1)
    rstd = (x.double().square().mean(1) + 1e-5).rsqrt().float()
    ds = ds if add else None
    dx, dw = L.rms_norm_backward(dy, x, w, rstd, dsum=ds)
    dt, size, want_w, size_w = reference_backward(dy, x, w, rstd, ds)
    within(dx, dt, size * (rms_chain(D) + 6) * U + dt.abs() * half(dtype) * 1.01 + 2.0 ** -133)
    # Rows of a thread, the groups of a workgroup, the workgroups by sixteens.
    within(dw, want_w, size_w * (M / 256 + 64 + 16 + 16 + 4) * U)
    if not add:
        same = L.rms_norm_backward(dy, x, None, rstd)
        ones = L.rms_norm_backward(dy, x, torch.ones_like(w), rstd)
        assert torch.equal(same[0], ones[0]) and torch.equal(same[1], ones[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_strides(gpu, dtype):
    x, ds, w = inputs(50, 333, dtype, 9, 340)
    dy = rows(50, 333, dtype, gen(4), 0.1, 335)
    rstd = (x.double().square().mean(1) + 1e-5).rsqrt().float()
    got = L.rms_norm_backward(dy, x, w, rstd, dsum=ds)
    want = L.rms_norm_backward(dy.contiguous(), x.contiguous(), w, rstd, dsum=ds.contiguous())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gradient_by_differences(gpu):
    """d(sum y c) / dx, and / dweight, by central differences of the 64-bit form.
    Their own error is h^2 / 6 of the third derivative, here below 1e-7."""
    g = gen(11)
    x, r, w = (torch.randn(3, 20, generator=g, device="cuda") for _ in range(3))
    w = w[0]
    c = torch.randn(3, 20, generator=g, device="cuda")
    _, t, rstd = L.rms_norm(x, w, residual=r, return_stats=True)
    dx, dw = L.rms_norm_backward(c, t, w, rstd)
    f = lambda x, w: float((rms(x, w, 1e-5, r)[0] * c.double()).sum())
    h = 1e-4
    for i, j in ((0, 0), (1, 7), (2, 19)):
        d = torch.zeros_like(x, dtype=torch.float64)
        d[i, j] = h
        want = (f(x.double() + d, w) - f(x.double() - d, w)) / (2 * h)
        assert abs(float(dx[i, j]) - want) < 1e-5
        e = torch.zeros_like(w, dtype=torch.float64)
        e[j] = h
        want = (f(x, w.double() + e) - f(x, w.double() - e)) / (2 * h)
        assert abs(float(dw[j]) - want) < 1e-5


def test_streams_and_graph(gpu):
    """Two streams at once, and a captured step replayed on new inputs."""
    x, r, w = inputs(500, 1000, torch.bfloat16, 12)
    dy = rows(500, 1000, torch.bfloat16, gen(13))
    def step():
        q, t, rstd = L.rms_norm_fp8(x, w, residual=r, return_stats=True)
        return (q.codes, q.scales, t, *L.rms_norm_backward(dy, t, w, rstd, dsum=r))
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (20, 21, 22):
        x2, r2, _ = inputs(500, 1000, torch.bfloat16, seed)
        x.copy_(x2)
        r.copy_(r2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals(gpu):
    x, r, w = inputs(8, 64, torch.float32, 14)
    rstd = torch.ones(8, device="cuda")
    for bad in (lambda: L.rms_norm(x.double()), lambda: L.rms_norm(x.half()), lambda: L.rms_norm(x, w.bfloat16()),
                lambda: L.rms_norm(x.cpu()), lambda: L.rms_norm_backward(x, x, w, None),
                lambda: L.rms_norm(x, residual=r.cpu())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: L.rms_norm(x, w[:-1]), lambda: L.rms_norm(x, residual=r[:-1]), lambda: L.rms_norm(x, residual=r.bfloat16()),
                lambda: L.rms_norm(x.t()), lambda: L.rms_norm(x, sum_out=r), lambda: L.rms_norm(x, residual=r, sum_out=r[:4]),
                lambda: L.rms_norm_backward(x[:4], x, w, rstd), lambda: L.rms_norm_backward(x, x, w, rstd[:4]),
                lambda: L.rms_norm_backward(x, x, w, rstd, dsum=r[:, :32]),
                lambda: L.rms_norm(x, residual=r, sum_out=torch.zeros_like(r).requires_grad_())):
        with pytest.raises(ValueError):
            bad()
    buf = torch.zeros(9, 64, device="cuda")
    for bad in (lambda: L.rms_norm(x, eps=-1.0), lambda: L.rms_norm(x, eps=float("nan")),
                lambda: L.rms_norm(buf[:-1], residual=r, sum_out=buf[1:]), lambda: L.rms_norm(x[:, :0])):
        with pytest.raises(_lib.NflowError):
            bad()
