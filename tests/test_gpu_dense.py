"""The bf16 / fp32 linear layer against its formula in 64 bits, forward and
backward: sizes around every tile, odd rows and strides, empty ones, results
known exactly, infinities, results in place, streams and captured graphs."""
import ctypes as C

import pytest
import torch

from neuroflow_amd import _lib, dense
from residual_reference import DTYPES, U, act, act_bound, gen, half, rows, within
from residual_reference import dense as product, dense_bound

pytestmark = pytest.mark.gpu
# (M, K, N): one row to thousands, odd everything; CUTS are the least that take every
# kernel and every way of dealing its tiles out, forward and backward (test_every_cut_is_met).
CUTS = [(33, 200, 4100), (33, 1025, 5003), (33, 2050, 3000), (33, 5003, 1537), (72, 72, 4100), (72, 130, 12000), (72, 4100, 72),
        (130, 72, 12000), (130, 12000, 72), (200, 33, 4100), (200, 1000, 8192), (200, 1025, 3000), (200, 1300, 4100),
        (200, 4100, 33), (200, 4100, 1300), (200, 8192, 1000), (257, 4100, 12000), (257, 12000, 4100), (1000, 1000, 1537),
        (1000, 1025, 4100), (1000, 4100, 1025), (1025, 33, 5003), (1025, 200, 3000), (1025, 3000, 200), (1025, 4100, 1000),
        (1025, 5003, 33), (1300, 200, 4100), (1537, 33, 5003), (1537, 5003, 33), (2050, 33, 3000), (2050, 3000, 33),
        (3000, 257, 8192), (4100, 72, 72), (8192, 200, 1000), (12000, 4100, 257), (65536, 1000, 1000), (40000, 1280, 2000), (40000, 2000, 1280),
        (200, 4100, 2050), (200, 2050, 4100), (4100, 2050, 200),
        (42, 64, 2792), (60, 512, 80), (64, 8192, 64), (495, 768, 118), (1000, 100, 100)]   # few steps to share
SIZES = [(1, 1, 1), (1, 4096, 4096), (2, 7, 3), (5, 100, 33), (16, 64, 16), (17, 200, 130), (33, 513, 64), (64, 31, 257),
         (65, 64, 64), (66, 1, 65), (100, 1000, 20), (129, 65, 127), (200, 2021, 301), (257, 128, 1000), (300, 8192, 136),
         (1000, 33, 1), (1537, 200, 1001), (2200, 96, 2056), (4099, 72, 2050), (2100, 2100, 40), (70, 2100, 2100),
         (4096, 256, 4096), (1, 16384, 100), (7, 16391, 65), (20, 8192, 1000)]


def weight(N, K, dtype, g, stride=None):
    w = (2 * torch.rand(N, K, generator=g, device="cuda") - 1) / K ** 0.5
    if stride is None:
        return w.to(dtype)
    buf = torch.full((N, stride), float("nan"), device="cuda", dtype=dtype)
    buf[:, :K] = w.to(dtype)
    return buf[:, :K]


def operands(M, K, N, dtype, seed, extra=(None, None, None)):
    g = gen(seed)
    return (rows(M, K, dtype, g, 1.0, extra[0] and K + extra[0]), weight(N, K, dtype, g, extra[1] and K + extra[1]),
            0.2 * torch.randn(N, generator=g, device="cuda"), rows(M, N, dtype, g, 0.5, extra[2] and N + extra[2]))


def check_forward(y, x, W, b, r, kind, pre=None):
    z, mag = product(x, W, b, r)
    zb = dense_bound(mag, x.shape[1], x.dtype)
    want = act(z, kind)[0]
    within(y, want, act_bound(z, zb, kind) + want.abs() * half(x.dtype) * 1.01 + 2.0 ** -133)
    if pre is not None:
        within(pre, z, zb + z.abs() * half(x.dtype) * 1.01 + 2.0 ** -133)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", SIZES)
def test_forward(gpu, M, K, N, dtype):
    x, W, b, r = operands(M, K, N, dtype, M + K + N)
    y, pre = dense.linear(x, W, b, "gelu", residual=r, return_pre=True)
    assert y.dtype == pre.dtype == dtype and y.shape == (M, N)
    check_forward(y, x, W, b, r, "gelu", pre)
    check_forward(dense.linear(x, W, None, "relu", residual=r), x, W, None, r, "relu")
    check_forward(dense.linear(x, W, b), x, W, b, None, "none")
    check_forward(dense.linear(x, W), x, W, None, None, "none")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(3, 50, 40), (70, 130, 90), (150, 64, 200), (700, 320, 384), (150, 200, 136), (1000, 72, 520)])
@pytest.mark.parametrize("extra", [(1, None, None), (None, 3, 1), (8, 8, 8), (5, 7, 9)])
def test_strides(gpu, M, K, N, dtype, extra):
    """Rows apart at any element alignment, with NaN between them."""
    x, W, b, r = operands(M, K, N, dtype, 3, extra)
    y = dense.linear(x, W, b, "gelu", residual=r)
    check_forward(y, x, W, b, r, "gelu")
    odd = torch.zeros(M, N + 3, device="cuda", dtype=dtype)
    dense.linear(x, W, b, "gelu", residual=r, out=odd[:, 1:N + 1])
    assert torch.equal(odd[:, 1:N + 1], y) and not bool(odd[:, 0].any()) and not bool(odd[:, N + 1:].any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 300, 50), (40, 100, 64), (100, 65, 30), (300, 700, 520), (2050, 96, 2050)])
def test_exact(gpu, M, K, N, dtype):
    """Whole numbers whose sums fit fp32: every result is known.  In fp32 of 17
    bits, which take all three parts of an operand, against at most 60 ones a row."""
    g = gen(M)
    if dtype == torch.bfloat16:
        x = torch.randint(-8, 9, (M, K), generator=g, device="cuda").float()
        W = torch.randint(-8, 9, (N, K), generator=g, device="cuda").float()
    else:
        x = torch.randint(-2 ** 17, 2 ** 17, (M, K), generator=g, device="cuda").float()
        W = torch.randint(-1, 2, (N, K), generator=g, device="cuda").float()
        W[:, 60:] = 0
        W = W[:, torch.randperm(K, generator=g, device="cuda")]
    b = torch.randint(-100, 101, (N,), generator=g, device="cuda").float()
    r = torch.randint(-100, 101, (M, N), generator=g, device="cuda").float()
    want = (x.double() @ W.double().t() + b.double() + r.double())
    got = dense.linear(x.to(dtype), W.to(dtype), b, residual=r.to(dtype))
    assert torch.equal(got, want.to(dtype))
    if dtype == torch.float32:                                 # the other operand of 17 bits
        got = dense.linear(W, x)
        assert torch.equal(got, (W.double() @ x.double().t()).float())
    # The backward products of the same kind of numbers.
    dy = torch.randint(-1, 2, (M, N), generator=g, device="cuda").float()
    if dtype == torch.float32:
        dy[60:] = 0
        dy[:, 60:] = 0
        W = torch.randint(-2 ** 17, 2 ** 17, (N, K), generator=g, device="cuda").float()
    dx, dW, db, dz = dense.linear_backward(dy.to(dtype), x.to(dtype), W.to(dtype))
    assert torch.equal(dx, (dy.double() @ W.double()).to(dtype))
    assert torch.equal(dW, (dy.double().t() @ x.double()).to(dtype))
    assert torch.equal(db, dy.double().sum(0).float())


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_axes_and_empty_sizes(gpu, dtype):
    x, W, b, r = operands(24, 96, 40, dtype, 4)
    want = dense.linear(x, W, b, residual=r)
    got = dense.linear(x.view(2, 3, 4, 96), W, b, residual=r.view(2, 3, 4, 40))
    assert got.shape == (2, 3, 4, 40) and torch.equal(got.view(24, 40), want)
    dx, dW, db, dz = dense.linear_backward(got, x.view(2, 3, 4, 96), W)
    flat = dense.linear_backward(want, x, W)
    assert dx.shape == (2, 3, 4, 96) and torch.equal(dx.view(24, 96), flat[0]) and torch.equal(dW, flat[1])
    assert dense.linear(x[:0], W, b).shape == (0, 40) and dense.linear(x, W[:0]).shape == (24, 0)
    for m in (24, 200):                                        # a sum over nothing
        rr = rows(m, 40, dtype, gen(2))
        y = dense.linear(torch.empty(m, 0, device="cuda", dtype=dtype), W[:, :0].contiguous(), b, "relu", residual=rr)
        within(y, (b.double() + rr.double()).clamp(min=0), (b.abs() + rr.double().abs()) * (2 * U + half(dtype)))
    dx, dW, db, dz = dense.linear_backward(want[:0], x[:0], W)
    assert dx.shape == (0, 96) and not bool(dW.any()) and not bool(db.any()) and dW.shape == W.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 64, 40), (80, 64, 40), (300, 513, 260)])
def test_out_is_the_residual(gpu, M, K, N, dtype):
    x, W, b, r = operands(M, K, N, dtype, 5)
    want = dense.linear(x, W, b, residual=r)
    version = r._version
    y = dense.linear(x, W, b, residual=r, out=r)
    assert y is r and torch.equal(r, want) and r._version == version + 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [2, 70, 300])
def test_infinities_stay_in_their_rows(gpu, dtype, M):
    """A row of x with an infinity or a NaN spoils its own results alone, a row
    of W its column, and rows past the last reach nothing."""
    K, N = 200, 150
    x, W, b, r = operands(M, K, N, dtype, 6)
    want = dense.linear(x, W, b, residual=r)
    x2, W2 = x.clone(), W.clone()
    x2[1, 199] = float("inf")
    W2[149, 0] = float("nan")
    got = dense.linear(x2, W2, b, residual=r)
    rest = torch.ones(M, N, dtype=torch.bool, device="cuda")
    rest[1], rest[:, 149] = False, False
    assert torch.equal(got[rest], want[rest]) and not bool(torch.isfinite(got[~rest]).any())
    # The largest finite values are no infinities to the parts of an operand.
    big = torch.finfo(torch.float32).max if dtype == torch.float32 else torch.finfo(dtype).max
    x3, W3 = torch.zeros(M, 8, device="cuda", dtype=dtype), torch.zeros(3, 8, device="cuda", dtype=dtype)
    x3[0, 3], W3[:, 3] = big, 0.5
    got = dense.linear(x3, W3)
    assert torch.equal(got[0], torch.full((3,), big * 0.5, device="cuda", dtype=dtype)) and not bool(got[1:].any())


@pytest.mark.parametrize("M,K,N", [(1, 300, 50), (80, 256, 64), (600, 256, 512)])
@pytest.mark.parametrize("exponent", [-112, -124, -130])
def test_tiny_operands(gpu, M, K, N, exponent):
    """fp32 operands whose last parts are subnormals of bf16, whose step is 2^-133:
    each operand is off by at most half of it."""
    g = gen(M)
    x = torch.randn(M, K, generator=g, device="cuda") * 2.0 ** exponent
    W = torch.randn(N, K, generator=g, device="cuda") * 2.0 ** 20
    for a, b in ((x, W), (W, x)):
        z, mag = product(a, b)
        tiny = 2.0 ** -134 * (a.double().abs().sum(1)[:, None] + b.double().abs().sum(1)[None, :])
        within(dense.linear(a, b), z, dense_bound(mag, K, torch.float32) + z.abs() * half(torch.float32) * 1.01 + tiny)


@pytest.mark.parametrize("M", [1, 40])
def test_rows_far_apart(gpu, M):
    """Strides that the tiled product of bf16 does not take, in whole 16-byte groups,
    and rows as long."""
    g, apart = gen(M), 2 ** 21
    x, W = (torch.zeros(n, apart, device="cuda", dtype=torch.bfloat16) for n in (M, 40))
    for t in (x, W):
        t[:, :64] = torch.randint(-8, 9, (len(t), 64), generator=g, device="cuda")
    xd, Wd = x[:, :64].double(), W[:, :64].double()
    want = (xd @ Wd.t()).to(torch.bfloat16)
    assert torch.equal(dense.linear(x[:, :64], W[:, :64]), want)
    assert torch.equal(dense.linear(x, W), want)
    dy = torch.randint(-1, 2, (M, 40), generator=g, device="cuda").bfloat16()
    for c in (64, apart):
        dx, dW, _, _ = dense.linear_backward(dy, x[:, :c], W[:, :c])
        assert torch.equal(dx[:, :64], (dy.double() @ Wd).to(torch.bfloat16)) and not bool(dx[:, 64:].any())
        assert torch.equal(dW[:, :64], (dy.double().t() @ xd).to(torch.bfloat16)) and not bool(dW[:, 64:].any())


def reference_backward(dy, x, W, kind, pre, dtype):
    """The formula's gradients with dz as the products take it (rounded), and
    their terms' magnitudes; dz before that."""
    full = dy.double() if kind == "none" else dy.double() * act(pre.double(), kind)[1]
    dz = full.to(dtype).double()
    return full, dz @ W.double(), dz.abs() @ W.double().abs(), dz.t() @ x.double(), dz.t().abs() @ x.double().abs()


@pytest.mark.parametrize("kind", ["none", "relu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", SIZES + [(8192, 130, 66), (9000, 256, 256)])
def test_backward(gpu, M, K, N, dtype, kind):
    x, W, _, _ = operands(M, K, N, dtype, M * 3 + K + N)
    g = gen(M)
    dy = rows(M, N, dtype, g, 0.1)
    pre = None if kind == "none" else (3 * torch.randn(M, N, generator=g, device="cuda")).to(dtype)
    dx, dW, db, dz = dense.linear_backward(dy, x, W, None if kind == "none" else kind, pre=pre)
    assert dx.dtype == dW.dtype == dz.dtype == dtype and db.dtype == torch.float32
    full, want_x, mag_x, want_w, mag_w = reference_backward(dy, x, W, kind, pre, dtype)
    # GELU's slope is formed from terms of up to 36 by 12 roundings and the exponent's.
    slope = {"none": 0.0, "relu": 0.0, "gelu": 2.0 ** -16}[kind]
    within(dz, full, full.abs() * half(dtype) * 1.01 + dy.double().abs() * slope + 2.0 ** -133)
    # dz may fall to the other side of a rounding than the reference's: once a step of each.
    flips = 0.0 if kind == "none" else 2 * half(dtype) + slope
    within(dx, want_x, dense_bound(mag_x, N, dtype) + mag_x * flips + (dy.double().abs() @ W.double().abs()) * slope +
           want_x.abs() * half(dtype) * 1.01 + 2.0 ** -133)
    within(dW, want_w, dense_bound(mag_w, M, dtype) + mag_w * flips + (dy.double().abs().t() @ x.double().abs()) * slope +
           want_w.abs() * half(dtype) * 1.01 + 2.0 ** -133)
    within(db, full.sum(0), full.abs().sum(0) * (M / 8 + 300) * U + dy.double().abs().sum(0) * slope)
    if kind == "none":
        assert dz is dy or dz.data_ptr() == dy.data_ptr()
    # The products of the rounded dz that came back, without that allowance.
    same = dense.linear_backward(dz, x, W)
    assert torch.equal(same[0], dx) and torch.equal(same[1], dW)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(37, 50, 41), (300, 129, 250), (203, 136, 200), (1003, 520, 72)])
@pytest.mark.parametrize("extra", [(1, 3, 5), (8, 16, 8)])
@pytest.mark.parametrize("apart", [2, 8])
def test_backward_strides(gpu, M, K, N, dtype, extra, apart):
    x, W, _, pre = operands(M, K, N, dtype, 8, extra)
    dy = rows(M, N, dtype, gen(9), 0.1, N + apart)
    full, want_x, mag_x, want_w, mag_w = reference_backward(dy, x, W, "none", None, dtype)
    dx, dW, db, _ = dense.linear_backward(dy, x, W)
    within(dx, want_x, dense_bound(mag_x, N, dtype) + want_x.abs() * half(dtype) * 1.01 + 2.0 ** -133)
    within(dW, want_w, dense_bound(mag_w, M, dtype) + want_w.abs() * half(dtype) * 1.01 + 2.0 ** -133)
    within(db, full.sum(0), full.abs().sum(0) * (M / 8 + 300) * U)
    got = dense.linear_backward(dy, x, W, "gelu", pre=pre)
    want = dense.linear_backward(dy.contiguous(), x.contiguous(), W.contiguous(), "gelu", pre=pre.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gelu_gradient_far_out(gpu, dtype):
    """Slopes at 0, where GELU is 0 or 1, at the largest values, and a NaN."""
    z = torch.tensor([[0.0, -0.0, 1.0, -1.0, 8.0, -8.0, 60.0, -60.0, 1e4, -1e4, 1e30, -1e30, 3e38, -3e38, float("nan")]],
                     device="cuda").to(dtype)
    N = z.shape[1]
    dy = torch.ones_like(z)
    W = torch.zeros(N, 4, device="cuda", dtype=dtype)
    dz = dense.linear_backward(dy, torch.zeros(1, 4, device="cuda", dtype=dtype), W, "gelu", pre=z)[3]
    want = torch.where(z.double().abs() > 50, (z > 0).double(), act(z.double().clamp(-50, 50), "gelu")[1])
    within(dz[:, :-1], want[:, :-1], want[:, :-1].abs() * half(dtype) * 1.01 + 2.0 ** -20)
    assert bool(torch.isnan(dz[0, -1]))
    dz = dense.linear_backward(dy, torch.zeros(1, 4, device="cuda", dtype=dtype), W, "relu", pre=z)[3]
    assert torch.equal(dz[:, :-1], (z > 0).to(dtype)[:, :-1]) and bool(torch.isnan(dz[0, -1]))


def test_gradient_by_differences(gpu):
    """d(sum y c) by central differences of the 64-bit form: their error is h^2
    / 6 of a third derivative below 10."""
    x, W, b, r = operands(5, 12, 9, torch.float32, 15)
    c = torch.randn(5, 9, generator=gen(16), device="cuda")
    _, pre = dense.linear(x, W, b, "gelu", residual=r, return_pre=True)
    got = dense.linear_backward(c, x, W, "gelu", pre=pre)
    f = lambda x, W, b, r: float((act(x @ W.t() + b + r, "gelu")[0] * c.double()).sum())
    h, at = 1e-4, [t.double() for t in (x, W, b, r)]
    for which, place in ((0, (2, 3)), (0, (4, 11)), (1, (0, 0)), (1, (8, 5)), (2, (4,)), (3, (1, 7))):
        up, down = [t.clone() for t in at], [t.clone() for t in at]
        up[which][place] += h
        down[which][place] -= h
        want = (f(*up) - f(*down)) / (2 * h)
        assert abs(float(got[which][place]) - want) < 2e-5 * max(1, abs(want)), (which, place)


def test_same_bits_streams_and_graph(gpu):
    x, W, b, r = operands(700, 1000, 520, torch.bfloat16, 17)
    dy = rows(700, 520, torch.bfloat16, gen(18), 0.1)
    def step():
        y, pre = dense.linear(x, W, b, "gelu", residual=r, return_pre=True)
        one = dense.linear(x[:1], W, b, residual=r[:1])
        return (y, pre, one, *dense.linear_backward(dy, x, W, "gelu", pre=pre))
    want = step()
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (20, 21, 22):
        x2, _, _, r2 = operands(700, 1000, 520, torch.bfloat16, seed)
        x.copy_(x2)
        r.copy_(r2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_every_cut_is_met(gpu):
    met = set()
    kernel, groups = C.c_int(), C.c_int()
    for M, K, N in SIZES + CUTS:
        for dt in (0, 1):
            for form, size in enumerate(((M, N, K), (M, K, N), (N, K, M), (M, N, K))):
                assert _lib.lib().nflow_debug_dense_cut(form, *size, dt, C.byref(kernel), C.byref(groups)) == _lib.OK
                met.add((form, dt, kernel.value, groups.value > 0))
    want = {(0, dt, 0, False) for dt in (0, 1)}                         # few rows
    for form in range(3):
        want |= {(form, 0, k, shared) for k in (1, 3, 5) for shared in (False, True)}
        want |= {(form, 1, k, False) for k in (1, 2, 3, 4, 5)} | {(form, 1, k, True) for k in (1, 2, 4, 5)}
    want |= {(3, 0, k, True) for k in (1, 3, 5)}
    assert want <= met, sorted(want - met)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", CUTS)
def test_cuts(gpu, M, K, N, dtype):
    """Every kernel, forward and backward, on whole numbers (every result known)
    and on operands that are, in bf16, 16-byte aligned in rows of their own stride."""
    g = gen(M)
    up = lambda n: (n + 7) // 8 * 8
    def whole(rows, cols, lo, hi, keep=None):
        buf = torch.full((rows, up(cols)), float("nan"), device="cuda", dtype=dtype)
        v = torch.randint(lo, hi, (rows, cols), generator=g, device="cuda").float()
        if keep is not None:                                             # a few columns alone are not zero
            v[:, torch.randperm(cols, generator=g, device="cuda")[keep:]] = 0
        buf[:, :cols] = v
        return buf[:, :cols]
    few = 60 if dtype == torch.float32 else None
    top = 2 ** 17 if dtype == torch.float32 else 3
    x, W = whole(M, K, -top, top), whole(N, K, -1, 2, few)
    y, pre = dense.linear(x, W, None, "relu", return_pre=True)
    want = x.double() @ W.double().t()
    assert torch.equal(pre, want.to(dtype)) and torch.equal(y, want.clamp(min=0).to(dtype))
    dy = whole(M, N, -1, 2, few)
    if few is not None:
        dy[torch.randperm(M, generator=g, device="cuda")[few:]] = 0
    W = whole(N, K, -top, top)
    dx, dW, db, dz = dense.linear_backward(dy, x, W)
    assert torch.equal(dx, (dy.double() @ W.double()).to(dtype))
    assert torch.equal(dW, (dy.double().t() @ x.double()).to(dtype))
    assert torch.equal(db, dy.double().sum(0).float())
    again = dense.linear_backward(dy.contiguous(), x.contiguous(), W.contiguous())
    assert all(torch.equal(a, b) for a, b in zip((dx, dW, db), again))


def test_refusals(gpu):
    x, W, b, r = operands(8, 64, 32, torch.float32, 19)
    for bad in (lambda: dense.linear(x.half(), W.half()), lambda: dense.linear(x, W.bfloat16()), lambda: dense.linear(x, W, b.bfloat16()),
                lambda: dense.linear(x.cpu(), W.cpu()), lambda: dense.linear(x, W, residual=r.cpu()),
                lambda: dense.linear_backward(r, x, W, "gelu"), lambda: dense.linear_backward(r, x.bfloat16(), W)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: dense.linear(x, W[:, :-1]), lambda: dense.linear(x, W.t()), lambda: dense.linear(x, W, b[:-1]),
                lambda: dense.linear(x, W, residual=r[:4]), lambda: dense.linear(x, W, residual=r.bfloat16()),
                lambda: dense.linear(x, W, activation="tanh"), lambda: dense.linear(x, W, out=r[:4]), lambda: dense.linear(x, W[0]),
                lambda: dense.linear_backward(r, x[:4], W), lambda: dense.linear_backward(r, x, W[:-1]),
                lambda: dense.linear_backward(r, x, W, None, pre=r), lambda: dense.linear_backward(r, x, W, "relu", pre=r[:4]),
                lambda: dense.linear(x, W, out=r.clone().requires_grad_())):
        with pytest.raises(ValueError):
            bad()
    buf = torch.zeros(9, 64, device="cuda")
    wide = torch.zeros(64, 64, device="cuda")
    for bad in (lambda: dense.linear(buf[:8], wide, out=buf[1:]), lambda: dense.linear(buf[:8], wide, out=buf[:8]),
                lambda: dense.linear(x, wide, out=wide[:8]), lambda: dense.linear(x, wide, residual=buf[:8], out=buf[1:])):
        with pytest.raises(_lib.NflowError):
            bad()
