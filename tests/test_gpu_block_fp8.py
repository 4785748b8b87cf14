"""128-block FP8: the quantise bit for bit against the oracle's codec, the
products and gradients against the formulas in 64 bits
(tests/block_reference.py; its bounds are derived there)."""
import numpy as np
import pytest
import torch

import block_reference as R
from neuroflow_amd import _lib
from neuroflow_amd import block_fp8 as B
from neuroflow_amd import norm as L
from neuroflow_amd import workloads as WL

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
F32 = torch.float32


def _x(seed, M, K, dtype=F32):
    x = (WL.normal(seed, (M, K)) * np.exp(WL.normal(seed + 1, (M, 1)))).astype(np.float32)
    t = torch.from_numpy(x).cuda().to(dtype)
    return t, t.float().cpu().numpy()


def _same(q, want, k):
    codes, scales = want
    assert q.k == k and q.codes.shape == codes.shape and q.scales.shape == scales.shape
    got = q.scales.cpu().numpy()
    assert np.array_equal(got.view(np.uint32), scales.view(np.uint32)), "scales"
    assert np.array_equal(q.codes.cpu().numpy(), codes), "codes"


# ---- quantise -------------------------------------------------------------------

SHAPES = [(1, 1), (1, 128), (1, 4096), (2, 127), (3, 129), (17, 1000), (127, 255), (128, 128), (129, 130), (130, 2021),
          (300, 64), (515, 7), (2000, 384)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K", SHAPES)
def test_quantise(gpu, M, K, dtype):
    t, x = _x(200 + M + K, M, K, dtype)
    rows, cols = R.quantise(x), R.quantise(np.ascontiguousarray(x.T))
    _same(B.quantise(t), rows, K)
    _same(B.quantise_columns(t), cols, M)
    q, c = B.quantise_both(t)
    _same(q, rows, K)
    _same(c, cols, M)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantise_strided_rows(gpu, dtype):
    """Rows at odd offsets and strides of a wider tensor."""
    for off, K in ((1, 200), (3, 128), (5, 77), (8, 512)):
        t, x = _x(230 + off, 150, K + 11, dtype)
        rows = R.quantise(np.ascontiguousarray(x[:, off:off + K]))
        cols = R.quantise(np.ascontiguousarray(x[:, off:off + K].T))
        v = t[:, off:off + K]
        _same(B.quantise(v), rows, K)
        q, c = B.quantise_both(v)
        _same(q, rows, K)
        _same(c, cols, 150)


def test_quantise_edge_values(gpu):
    """Zero blocks, blocks below the least scale, ties, the capped range below
    2^-6, NaN beside numbers, NaN alone, infinities, the largest values."""
    x = WL.normal(240, (140, 300)).astype(np.float32)
    x[0] = 0.0
    x[1, :128] = 1e-37 * np.sign(x[1, :128])
    x[2, :128] = 5e-39
    x[3, :] = -0.0
    x[4, 3] = np.nan
    x[5, :128] = np.nan
    x[6, 7] = np.inf
    x[7, 9] = -np.inf
    x[8, 10], x[8, 11] = np.inf, np.nan
    x[9, :] = 3.4e38
    x[10, :128] = np.arange(128) * 0.5 * 2.0 ** -9       # scale 1 of a block with absmax 448
    x[10, 0] = 448.0
    x[11, :128] = 448.0 * 2.0 ** -126
    x[12, :128] = np.float32(448.0 * 2.0 ** -126) * np.float32(0.99)
    with np.errstate(invalid="ignore", over="ignore"):
        rows, cols = R.quantise(x), R.quantise(np.ascontiguousarray(x.T))
    t = torch.from_numpy(x).cuda()
    _same(B.quantise(t), rows, 300)
    _same(B.quantise_columns(t), cols, 140)
    q, c = B.quantise_both(t)
    _same(q, rows, 300)
    _same(c, cols, 140)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (127, 129), (300, 1000), (768, 256), (5, 513)])
def test_quantise_weight(gpu, N, K, dtype):
    t, W = _x(250 + N + K, N, K, dtype)
    want = R.quantise_weight(W)
    _same(B.quantise_weight(t), want, K)
    w, wt = B.quantise_weight(t, transposed=True)
    _same(w, want, K)
    codes = np.zeros((K, 128 * R.blocks(N)), np.uint8)
    codes[:, :N] = want[0][:, :K].T
    _same(wt, (codes, np.ascontiguousarray(want[1].T)), N)


def test_quantise_past_32_bit_offsets(gpu):
    M, K = (1 << 20) + 70, 4096
    x = torch.zeros(M, K, dtype=BF16, device="cuda")
    t, tail = _x(260, 70, K, BF16)
    x[-70:] = t
    q = B.quantise(x)
    small = B.quantise(t)
    assert torch.equal(q.codes[-70:], small.codes) and torch.equal(q.scales[:, -70:], small.scales)
    del q
    _, c = B.quantise_both(x)
    # The last column block starts at row 2^20, where the tail's rows begin.
    want = R.quantise(np.ascontiguousarray(tail.T))
    assert np.array_equal(c.codes[:, 1 << 20:].cpu().numpy(), want[0])
    assert np.array_equal(c.scales[-1].cpu().numpy(), want[1][0])


# ---- products ---------------------------------------------------------------------

def _operands(seed, M, N, K, wide=False):
    _, x = _x(seed, M, K)
    W = WL.uniform(seed + 5, (N, K), -0.2, 0.2).astype(np.float32)
    a = R.quantise(x)
    w = R.quantise(W) if wide else R.quantise_weight(W)
    return a, w


def _block(q, k):
    return B.BlockFp8(torch.from_numpy(q[0]).cuda(), torch.from_numpy(q[1]).cuda(), k)


def _check(y, a, w, bias, act, K):
    want, mag = R.matmul(R.values(*a), R.values(*w), bias, act)
    tol = R.matmul_tol(mag, want, K, y.dtype == BF16)
    over = np.abs(y.double().cpu().numpy() - want) - tol
    assert (over <= 0).all(), f"{over.max():.3g} over its bound at {np.unravel_index(over.argmax(), over.shape)}"


# Single tokens, a few, the tile edges, many; odd widths and one value to many blocks of them.
PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 1000, 200), (1, 4096, 1024), (2, 65, 129), (7, 300, 1000), (16, 512, 512),
            (17, 130, 640), (33, 257, 385), (64, 64, 64), (65, 768, 256), (100, 48, 5000), (127, 129, 127),
            (128, 256, 128), (129, 1544, 300), (200, 1000, 1001), (255, 513, 257), (256, 256, 256), (300, 515, 4096),
            (513, 770, 384), (1000, 1000, 1000), (2049, 300, 130), (96, 96, 20000)]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_matmul(gpu, M, N, K, out):
    bias = WL.uniform(301, (N,), -1, 1).astype(np.float32)
    for wide in (False, True):
        a, w = _operands(300 + M + N + K, M, N, K, wide)
        if wide and N == 1:
            continue
        qa, qw = _block(a, K), _block(w, K)
        y = B.matmul(qa, qw, torch.from_numpy(bias).cuda(), "gelu", out)
        _check(y, a, w, bias, "gelu", K)
        assert torch.equal(B.matmul(qa, qw, torch.from_numpy(bias).cuda(), "gelu", out), y)
        y = B.matmul(qa, qw, out_dtype=out)
        _check(y, a, w, None, None, K)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(4096, 4096, 256), (4001, 4099, 300), (512, 1024, 8192), (65, 1000, 8200), (64, 2000, 8192),
                                   (1, 8192, 2048), (20000, 768, 256)])
def test_matmul_cuts(gpu, M, N, K, out):
    """Enough rows and columns for each tile, and few enough for splits over K."""
    bias = WL.uniform(305, (N,), -1, 1).astype(np.float32)
    for wide in (False, True):
        a, w = _operands(306 + M + N + K, M, N, K, wide)
        y = B.matmul(_block(a, K), _block(w, K), torch.from_numpy(bias).cuda(), "relu", out)
        _check(y, a, w, bias, "relu", K)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M", [1, 5, 40, 300])
def test_matmul_all_codes(gpu, M, out):
    """Every finite code in both operands, scales over many magnitudes."""
    K, N = 384, 200
    codes = np.array([c for c in range(256) if c & 0x7F != 0x7F], np.uint8)
    rng = np.random.default_rng(7)
    a = (rng.choice(codes, (M, K)), np.exp2(rng.uniform(-20, 20, (3, M))).astype(np.float32))
    w = (rng.choice(codes, (N, K)), np.exp2(rng.uniform(-20, 20, (3, 2))).astype(np.float32))
    _check(B.matmul(_block(a, K), _block(w, K), activation="relu", out_dtype=out), a, w, None, "relu", K)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M", [3, 70, 260])
def test_matmul_nonfinite_stays_in_its_row_and_column(gpu, M, out):
    K, N = 256, 300
    a, w = _operands(310, M, N, K)
    clean = B.matmul(_block(a, K), _block(w, K), out_dtype=out)
    a[0][1, 200] = 0x7F
    w[0][5, 3] = 0xFF
    y = B.matmul(_block(a, K), _block(w, K), out_dtype=out)
    assert torch.isnan(y[1]).all() and torch.isnan(y[:, 5]).all()
    rows, cols = [r for r in range(M) if r != 1], [c for c in range(N) if c != 5]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])


def test_matmul_empty(gpu):
    def e(rows, K):
        return B.BlockFp8(torch.empty(rows, 128 * R.blocks(K), dtype=torch.uint8, device="cuda"),
                          torch.empty(R.blocks(K), rows, device="cuda"), K)
    assert B.matmul(e(0, 128), e(4, 128)).shape == (0, 4)
    assert B.matmul(e(4, 128), e(0, 128)).shape == (4, 0)
    b = torch.tensor([1.0, -2.0, 3.0], device="cuda")
    for M in (2, 100):
        y = B.matmul(e(M, 0), e(3, 0), b, "relu", BF16)
        assert torch.equal(y.float(), b.clamp(min=0).expand(M, 3))
        y = B.linear(torch.zeros(M, 0, device="cuda"), B.BlockFp8(*e(3, 0)[:1], torch.empty(0, 1, device="cuda"), 0), b)
        assert torch.equal(y, b.expand(M, 3))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 4096, 4096), (1, 1000, 200), (2, 130, 1001), (3, 768, 256), (8, 64, 5000),
                                   (15, 300, 640), (16, 512, 128), (17, 512, 129), (33, 200, 1000), (64, 1024, 1024),
                                   (65, 300, 384), (500, 768, 256), (1001, 1001, 129)])
def test_linear(gpu, M, N, K, dtype):
    """linear is the matmul of the quantised rows, for every row count, type and stride."""
    t, x = _x(320 + M + N + K, M, K, dtype)
    W = WL.uniform(321, (N, K), -0.2, 0.2).astype(np.float32)
    w = R.quantise_weight(W)
    bias = WL.uniform(322, (N,), -1, 1).astype(np.float32)
    a = R.quantise(x)
    y = B.linear(t, _block(w, K), torch.from_numpy(bias).cuda(), "gelu")
    assert y.dtype == dtype
    _check(y, a, w, bias, "gelu", K)
    wide = torch.zeros(M, K + 3, dtype=dtype, device="cuda")
    wide[:, 1:1 + K] = t
    assert torch.equal(B.linear(wide[:, 1:1 + K], _block(w, K), torch.from_numpy(bias).cuda(), "gelu"), y)
    _check(B.linear(t.view(1, M, K), _block(w, K))[0], a, w, None, None, K)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [1, 4, 40])
def test_linear_nonfinite_rows(gpu, M, dtype):
    """A NaN makes its row NaN, an infinity too; the other rows keep their bits."""
    t, _ = _x(330, M + 2, 300, dtype)
    w = _block(R.quantise_weight(WL.uniform(331, (70, 300), -0.2, 0.2).astype(np.float32)), 300)
    clean = B.linear(t, w)
    t[0, 299], t[1, 5] = float("nan"), float("inf")
    y = B.linear(t, w)
    assert torch.isnan(y[:2]).all() and torch.equal(y[2:], clean[2:])


# ---- backward ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 300, 200), (5, 128, 128), (64, 768, 256), (129, 130, 131), (1000, 200, 77),
                                   (515, 385, 1000), (4099, 256, 300), (20000, 64, 96),
                                   (5003, 1544, 1000)])
def test_linear_backward(gpu, M, N, K, dtype):
    t, x = _x(340 + M + N + K, M, K, dtype)
    dyt, dy = _x(350 + M + N + K, M, N, dtype)
    W = WL.uniform(341, (N, K), -0.2, 0.2).astype(np.float32)
    _, xc = B.quantise_both(t)
    w, wt = B.quantise_weight(torch.from_numpy(W).cuda(), transposed=True)
    dx, dw, db = B.linear_backward(dyt, xc, wt)
    assert dx.dtype == dtype and dw.dtype == F32 and db.dtype == F32
    rows, cols = R.quantise(dy), R.quantise(np.ascontiguousarray(dy.T))
    _check(dx, rows, (wt.codes.cpu().numpy(), wt.scales.cpu().numpy()), None, None, N)
    _check(dw, cols, R.quantise(np.ascontiguousarray(x.T)), None, None, M)
    db64 = dy.astype(np.float64).sum(axis=0)
    tol = (M / 64 + 200) * R.U * np.abs(dy.astype(np.float64)).sum(axis=0) + 1e-30
    assert (np.abs(db.double().cpu().numpy() - db64) <= tol).all()
    again = B.linear_backward(dyt, xc, wt)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def test_linear_backward_against_differences(gpu):
    """The layer is linear in W's and x's values: differences of the 64-bit
    <q(dy), x W^T> along a direction are the gradients' inner products."""
    M, N, K = 50, 140, 90
    t, x = _x(360, M, K)
    dyt, dy = _x(361, M, N)
    _, xc = B.quantise_both(t)
    w, wt = B.quantise_weight(torch.from_numpy(WL.uniform(362, (N, K), -0.2, 0.2).astype(np.float32)).cuda(), True)
    dx, dw, _ = B.linear_backward(dyt, xc, wt)
    Wv = R.values(w.codes.cpu().numpy(), w.scales.cpu().numpy())[:, :K]
    xv = R.values(xc.codes.cpu().numpy(), xc.scales.cpu().numpy())[:, :M].T
    gr = R.values(*R.quantise(dy))[:, :N]
    gc = R.values(*R.quantise(np.ascontiguousarray(dy.T)))[:, :M].T
    vx, vw = WL.normal(363, (M, K)), WL.normal(364, (N, K))
    for got, f in (((dx.double().cpu().numpy() * vx).sum(), lambda e: (gr * ((xv + e * vx) @ Wv.T)).sum()),
                   ((dw.double().cpu().numpy() * vw).sum(), lambda e: (gc * (xv @ (Wv + e * vw).T)).sum())):
        want = (f(0.5) - f(-0.5)) / 1.0
        mag = max(np.abs(gr).sum() * np.abs(Wv).max() * np.abs(vx).max(), np.abs(gc).sum() * np.abs(xv).max() * np.abs(vw).max())
        assert abs(got - want) <= 300 * R.U * mag


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(17, 1, 1), (17, 129, 128), (64, 7, 100), (65, 33, 129), (100, 500, 200), (129, 4097, 90),
                                   (700, 130, 256), (2049, 1000, 300), (2100, 70, 512), (8200, 256, 500),
                                   (16384, 768, 256), (33000, 640, 120)])
def test_linear_is_the_product_of_the_codes(gpu, M, N, K, dtype):
    """Whichever kernel a size takes, linear gives the bits of quantise and
    matmul: rows of zeros, infinities and NaN, odd row strides, every activation."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    wide = (torch.randn(M, K + 5, device="cuda", generator=g) * torch.randn(M, 1, device="cuda", generator=g).exp()).to(dtype)
    w = B.quantise_weight(torch.randn(N, K, device="cuda", generator=g))
    bias = torch.randn(N, device="cuda", generator=g)
    for off in (0, 3):
        x = wide[:, off:off + K]
        x[M // 2] = 0
        x[M // 3, K // 2] = float("inf")
        x[M // 4, K - 1] = float("nan")
        x[M - 1, 0] = -1e30
        for b, act in ((None, "none"), (bias, "relu"), (bias, "gelu")):
            got, want = B.linear(x, w, b, act), B.matmul(B.quantise(x), w, b, act, out_dtype=dtype)
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(got.nan_to_num(nan=0.5), want.nan_to_num(nan=0.5))
    strided = wide.t().contiguous().t()[:, :K].contiguous().unsqueeze(0)
    assert torch.equal(B.linear(strided, w).nan_to_num(nan=0.5)[0],
                       B.matmul(B.quantise(strided[0]), w, out_dtype=dtype).nan_to_num(nan=0.5))


@pytest.mark.parametrize("M,N,K", [(40, 24, 32), (700, 48, 130), (3000, 150, 200), (65, 257, 300)])
def test_linear_backward_of_some_results(gpu, M, N, K):
    """Each result has the same bits whichever others the call is asked for."""
    import ctypes
    lib = _lib.lib()
    dy, _ = _x(640 + M, M, N)
    xc = B.quantise_columns(_x(641 + M, M, K)[0])
    _, wt = B.quantise_weight(_x(642 + M, N, K)[0], transposed=True)
    want = B.linear_backward(dy, xc, wt)
    need = ctypes.c_size_t()
    assert lib.nflow_fp8_block_linear_backward_workspace(M, N, K, _lib.DTYPE_F32, ctypes.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    for ask in range(1, 8):
        got = [torch.full_like(t, 7.0) for t in want]
        p = [t.data_ptr() if ask >> i & 1 else None for i, t in enumerate(got)]
        rc = lib.nflow_fp8_block_linear_backward(
            dy.data_ptr(), _lib.DTYPE_F32, M, N, N, xc.codes.data_ptr(), xc.scales.data_ptr(), wt.codes.data_ptr(),
            wt.scales.data_ptr(), K, p[0], K, p[1], p[2], ws.data_ptr(), need.value,
            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        for i in range(3):
            assert torch.equal(got[i], want[i] if ask >> i & 1 else torch.full_like(want[i], 7.0)), (ask, i)


def test_linear_backward_empty(gpu):
    w, wt = B.quantise_weight(torch.ones(30, 20, device="cuda"), transposed=True)
    xc = B.quantise_columns(torch.empty(0, 20, device="cuda"))
    dx, dw, db = B.linear_backward(torch.empty(0, 30, device="cuda"), xc, wt)
    assert dx.shape == (0, 20) and dw.shape == (30, 20) and not dw.any() and not db.any()


# ---- refusals, streams, graphs -----------------------------------------------------------

def test_refusals(gpu):
    x = torch.zeros(4, 300, device="cuda")
    q, w = B.quantise(x), B.quantise_weight(torch.zeros(200, 300, device="cuda"))
    with pytest.raises(TypeError):
        B.quantise(x.half())
    with pytest.raises(TypeError):
        B.quantise(x.cpu())
    with pytest.raises(ValueError):
        B.quantise(x.t())
    with pytest.raises(ValueError):
        B.linear(x[:, :299], w)
    with pytest.raises(ValueError):
        B.linear(x, w, torch.zeros(199, device="cuda"))
    with pytest.raises(ValueError):
        B.linear(x, q._replace(k=300))          # rows' scales where a weight's are due
    with pytest.raises(ValueError):
        B.linear(x, w, activation="tanh")
    with pytest.raises(ValueError):
        B.matmul(q._replace(k=301), w)
    with pytest.raises(ValueError):
        B.matmul(q._replace(codes=q.codes[:, :128].contiguous()), w)
    with pytest.raises(ValueError):
        B.matmul(w, q)                           # a weight's scales on the left
    with pytest.raises(TypeError):
        B.matmul(q, w, out_dtype=torch.float16)
    with pytest.raises(TypeError):
        B.matmul(q._replace(codes=q.codes.view(torch.int8)), w)
    with pytest.raises(ValueError):
        B.linear_backward(torch.zeros(4, 200, device="cuda"), B.quantise_columns(x[:3]),
                          B.quantise_weight(torch.zeros(200, 300, device="cuda"), True)[1])
    lib, p, s = _lib.lib(), q.codes.data_ptr(), q.scales.data_ptr()
    out = torch.empty(4, 200, device="cuda")
    args = [p, s, w.codes.data_ptr(), w.scales.data_ptr(), 1, 4, 200, 300, None, 0, out.data_ptr(), 0, 200, None, 0, 0]
    n = _lib.C.c_size_t()
    assert lib.nflow_fp8_block_matmul_workspace(4, 200, 300, 0, _lib.C.byref(n)) == 0
    ws = torch.empty(n.value + 1, dtype=torch.uint8, device="cuda")
    args[13], args[14] = ws.data_ptr(), n.value
    assert lib.nflow_fp8_block_matmul(*args) == 0
    for at, value in ((0, None), (1, None), (0, p + 1), (5, -1), (7, (1 << 22) + 1), (9, 3), (10, None), (11, 2), (12, 199)):
        bad = list(args)
        bad[at] = value
        assert lib.nflow_fp8_block_matmul(*bad) == _lib.INVALID_ARG, (at, value)
        assert b"fp8_block_matmul" in lib.nflow_last_error()
    need = _lib.C.c_size_t()
    assert lib.nflow_fp8_block_linear_workspace(100, 200, 300, 0, _lib.C.byref(need)) == 0 and need.value > 0
    x100, y = torch.zeros(100, 300, device="cuda"), torch.zeros(100, 200, device="cuda")
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    for have in (0, need.value - 1):
        assert lib.nflow_fp8_block_linear(x100.data_ptr(), 0, 100, 300, 300, args[2], args[3], 200, None, 0, y.data_ptr(),
                                          200, ws.data_ptr() if have else None, have, 0) == _lib.INVALID_ARG


def test_streams_do_not_share_scratch(gpu):
    """Two streams at once, each with its own operands, several times over."""
    K, N = 1024, 512
    ops = []
    for i in range(2):
        t, _ = _x(370 + i, 700, K, BF16)
        w, wt = B.quantise_weight(torch.from_numpy(WL.uniform(372 + i, (N, K), -0.2, 0.2).astype(np.float32)).cuda(), True)
        dy, _ = _x(374 + i, 700, N, BF16)
        xc = B.quantise_columns(t)
        ops.append((t, w, wt, dy, xc, B.linear(t, w), B.linear_backward(dy, xc, wt)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            t, w, wt, dy, xc, _, _ = ops[i]
            with torch.cuda.stream(st):
                got[i].append((B.linear(t, w), B.linear_backward(dy, xc, wt)))
    torch.cuda.synchronize()
    for i in range(2):
        for y, g in got[i]:
            assert torch.equal(y, ops[i][5]) and all(torch.equal(p, q) for p, q in zip(g, ops[i][6]))


@pytest.mark.parametrize("M", [1, 300])
def test_graph_replays(gpu, M):
    """A norm, a layer and their backward captured once, replayed on new
    inputs with eager calls between."""
    K, N = 512, 384
    x, _ = _x(380, M, K, BF16)
    dy, _ = _x(381, M, N, BF16)
    g, b = torch.ones(K, device="cuda"), torch.zeros(K, device="cuda")
    w, wt = B.quantise_weight(torch.from_numpy(WL.uniform(382, (N, K), -0.2, 0.2).astype(np.float32)).cuda(), True)

    def step():
        h, mean, rstd = L.layer_norm(x, g, b, return_stats=True)
        q, c = B.quantise_both(h)
        y = B.matmul(q, w, out_dtype=BF16)
        dh, dw, db = B.linear_backward(dy, c, wt)
        return (y, B.linear(h, w), dw, db, *L.layer_norm_backward(dh, x, g, mean, rstd))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.copy_(_x(383 + k, M, K, BF16)[0])
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))
