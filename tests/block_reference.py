"""64-bit statements of layer norm and the 128-block FP8 layer, for the tests.

Everything is float64 numpy from the formulas; the FP8 codes come from the
oracle's per-token quantise applied to each run of 128 values, so they are
compared bit for bit.
"""
import numpy as np

from oracle import oracle as O

U = 2.0 ** -24           # unit roundoff of fp32
U16 = 2.0 ** -8          # of bf16 (8 significant bits: half a unit in the last place of 1)
TINY = 448.0 * 2.0 ** -126


def blocks(n):
    return -(-n // 128)


def quantise(x):
    """(codes (M, 128 * blocks) uint8, scales (blocks, M) float32) of x (M, K) float32."""
    M, K = x.shape
    kb = blocks(K)
    P = np.zeros((M, kb * 128), np.float32)
    P[:, :K] = x
    q, s = O.quantise_per_token_fp8(P.reshape(M * kb, 128))
    q, s = np.array(q).reshape(M * kb, 128), np.array(s, np.float32).reshape(-1)
    amax = np.fmax.reduce(np.abs(P.reshape(M * kb, 128)), axis=1)
    tiny = np.nan_to_num(amax, nan=0.0) < TINY
    if tiny.any():
        s[tiny] = 1.0
        q[tiny] = O.e4m3_encode(P.reshape(M * kb, 128)[tiny].reshape(-1)).reshape(-1, 128)
    q = q.reshape(M, kb * 128)
    q[:, K:] = 0
    return q, np.ascontiguousarray(s.reshape(M, kb).T)


def quantise_weight(W):
    """(codes (N, 128 * blocks), scales (blocks, row blocks)) with a scale for every 128 x 128 block."""
    N, K = W.shape
    nb, kb = blocks(N), blocks(K)
    P = np.zeros((nb * 128, kb * 128), np.float32)
    P[:N, :K] = W
    q, s = O.quantise_per_token_fp8(P.reshape(nb, 128, kb, 128).transpose(0, 2, 1, 3).reshape(nb * kb, 128 * 128))
    q = np.array(q).reshape(nb, kb, 128, 128).transpose(0, 2, 1, 3).reshape(nb * 128, kb * 128)[:N]
    return np.ascontiguousarray(q), np.ascontiguousarray(np.array(s, np.float32).reshape(nb, kb).T)


def values(codes, scales):
    """float64 values of codes (R, 128 * blocks) with scales (blocks, R or row blocks)."""
    R = codes.shape[0]
    v = O.e4m3_decode(np.ascontiguousarray(codes).reshape(-1)).astype(np.float64).reshape(codes.shape)
    s = scales.astype(np.float64)
    if s.shape[1] != R:
        s = np.repeat(s, 128, axis=1)[:, :R]
    return v * np.repeat(s.T, 128, axis=1)


def activate(z, act):
    if act == "relu":
        return np.where(z < 0, 0.0, z)
    if act == "gelu":
        return z / (1.0 + np.exp(-2.0 * np.sqrt(2.0 / np.pi) * (z + 0.044715 * z ** 3)))
    return z


def matmul(A, W, bias=None, act=None):
    """(result, scale of its rounding: the sum of magnitudes)."""
    z, mag = A @ W.T, np.abs(A) @ np.abs(W).T
    if bias is not None:
        z, mag = z + bias, mag + np.abs(bias)
    return activate(z, act), mag


def matmul_tol(mag, y, K, bf16):
    """Bound on the product's error.  fp32: 128 products are summed, then one
    scaled sum per block joins (each operation within U of the sum of
    magnitudes), the activation's slope is below 1.13 and its own error a few
    U of y.  bf16: the FP8 instruction may lose 2^-12 of a block's sum of
    magnitudes, and the result is rounded to bf16."""
    t = 1.13 * (128 + 2 * blocks(K) + 6) * U * mag + 2.0 ** -20 * np.abs(y) + 1e-30
    return t + 1.13 * 2.0 ** -11 * mag + U16 * np.abs(y) * 1.01 if bf16 else t


def norm(x, w, b, eps):
    mean = x.mean(axis=1)
    rstd = 1.0 / np.sqrt(((x - mean[:, None]) ** 2).mean(axis=1) + eps)
    h = (x - mean[:, None]) * rstd[:, None]
    return h * (1.0 if w is None else w) + (0.0 if b is None else b), mean, rstd


def norm_tols(x, w, b, eps, y, rstd, bf16):
    """Bounds on (y, mean, rstd).  Sums over D run in chains of at most D / 64
    additions joined by at most 16 more, each within U: the mean is off by at
    most g = (D / 64 + 16) U of the mean magnitude; the deviations by that and
    a rounding; the variance by twice the relative error of the deviations
    against sigma plus g; rstd by half of it, and two roundings."""
    D = x.shape[1]
    g = (D / 64 + 16) * U
    dm = g * np.abs(x).mean(axis=1) + U * np.abs(x.mean(axis=1))
    dev = dm + 2 * U * np.abs(x - x.mean(axis=1, keepdims=True)).max(axis=1) + U * np.abs(x).max(axis=1)
    rel = 2 * dev * rstd + g + 6 * U                       # of the variance, then of rstd (an upper bound)
    h = (x - x.mean(axis=1, keepdims=True)) * rstd[:, None]
    aw = 1.0 if w is None else np.abs(w)
    ty = aw * (dev * rstd)[:, None] + aw * np.abs(h) * (rel + 4 * U)[:, None] + 3 * U * np.abs(y)
    if b is not None:
        ty = ty + U * np.abs(b)
    if bf16:
        ty = ty + U16 * 1.01 * np.abs(y)
    return ty + 1e-30, dm + 1e-30, rel * rstd


def norm_grad(dy, x, w, mean, rstd):
    D = x.shape[1]
    h = (x - mean[:, None]) * rstd[:, None]
    g = dy * (1.0 if w is None else w)
    c1, c2 = g.sum(axis=1, keepdims=True) / D, (g * h).sum(axis=1, keepdims=True) / D
    return rstd[:, None] * (g - c1 - h * c2), (dy * h).sum(axis=0), dy.sum(axis=0), h, g


def norm_grad_tols(dy, x, h, g, rstd, dx, bf16):
    """Bounds on (dx, dweight, dbias): h carries 3 U of itself and U of x rstd;
    row sums as in norm_tols; column sums run in chains of at most M / 64 + 64
    additions joined by at most 16."""
    M, D = x.shape
    gr, gc = (D / 64 + 16) * U, (M / 64 + 64 + 16) * U
    eh = 3 * U * np.abs(h) + 2 * U * np.abs(x) * rstd[:, None]
    mg, mgh = np.abs(g).mean(axis=1, keepdims=True), np.abs(g * h).mean(axis=1, keepdims=True)
    megh = (np.abs(g) * eh).mean(axis=1, keepdims=True)
    r = rstd[:, None]
    t = r * (4 * U * np.abs(g) + (gr + 4 * U) * mg + np.abs(h) * ((gr + 6 * U) * mgh + megh) + eh * mgh)
    if bf16:
        t = t + U16 * 1.01 * np.abs(dx)
    tw = gc * np.abs(dy * h).sum(axis=0) + (np.abs(dy) * (eh + U * np.abs(h))).sum(axis=0)
    return t + 1e-30, tw + 1e-30, gc * np.abs(dy).sum(axis=0) + 1e-30
