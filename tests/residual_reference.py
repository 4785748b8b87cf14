"""Plain 64-bit forms of include/nflow_residual.h's operators, and bounds of the
kernels' errors from their arithmetic."""
import math

import torch

U = 2.0 ** -24                     # half a step of fp32
C, C3 = math.sqrt(2 / math.pi), 0.044715
DTYPES = [torch.float32, torch.bfloat16]


def half(dtype):
    """The most that a rounding to dtype is off, relative to the value."""
    return torch.finfo(dtype).eps / 2


def rows(M, D, dtype, g, scale=1.0, stride=None):
    """Normal values, each row with a level of its own; stride: in rows that far apart."""
    x = torch.randn(M, D, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(M, 1, generator=g, device="cuda")) * scale
    if stride is None:
        return x.to(dtype)
    buf = torch.full((max(M, 1), stride), float("nan"), device="cuda", dtype=dtype)
    buf[:M, :D] = x.to(dtype)
    return buf[:M, :D]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, bound):
    """Every value no further from `want` than `bound` says (64 bits)."""
    assert got.shape == want.shape, (got.shape, want.shape)
    far = (got.double() - want).abs() - bound
    assert not bool(torch.isnan(far).any()), "NaN"
    worst = float(far.max()) if far.numel() else 0.0
    assert worst <= 0, f"{worst:.3e} past the bound, of values up to {float(want.abs().max()):.3e}"


def rms(x, weight, eps, residual=None):
    """y, t, rstd."""
    t = x.double() if residual is None else x.double() + residual.double()
    rstd = (t.square().mean(-1) + eps).rsqrt()
    y = t * rstd[..., None] * (1.0 if weight is None else weight.double())
    return y, t, rstd


def rms_chain(D):
    """Roundings on the way of a row's sum of squares: up to 16 or D / 256 in a
    thread, six across a wave and up to 16 across waves, the mean, eps."""
    return max(16, D // 256 + 1) + 24


def act(z, kind):
    """act(z) and its derivative."""
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "gelu":
        p = torch.sigmoid(2 * C * (z + C3 * z ** 3))
        return z * p, p + z * p * (1 - p) * 2 * C * (1 + 3 * C3 * z * z)
    return z, torch.ones_like(z)


def dense(x, W, bias=None, residual=None):
    """z and the sum of its terms' magnitudes, of 2-D operands."""
    z = x.double() @ W.double().t()
    mag = x.double().abs() @ W.double().abs().t()
    for term in (bias, residual):
        if term is not None:
            z = z + term.double()
            mag = mag + term.double().abs()
    return z, mag


def dense_bound(mag, K, dtype):
    """K + 4 additions that may each be off by a step of fp32; fp32 products from
    their six parts are off by 2^-26 and join six times."""
    return mag * (6 * K + 8 if dtype == torch.float32 else K + 4) * 2 * U


def act_bound(z, zb, kind):
    """What z's bound becomes behind the activation: its slope is at most 1.13,
    and GELU's exponent, up to 36 for |z| < 6, is off by two roundings of itself."""
    if kind != "gelu":
        return zb
    return 1.13 * zb + act(z, kind)[0].abs() * 2.0 ** -16 + 2.0 ** -40
