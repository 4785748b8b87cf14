"""Layer norm and the linear layer of 128-block FP8, as measurable cases.

A transformer or token-mixer block of 8-bit models is a norm, a quantise and a
matrix product; training it runs the same three backwards. Each case here is
one call of that path, through neuroflow_amd.norm and neuroflow_amd.block_fp8:

  norm         y, mean, rstd = layer norm over the last axis of x (M, D)
  norm_fp8     the same, y as E4M3 codes with a scale for every 128 features,
               the form the next product takes
  norm_grad    dx, dweight, dbias of the layer norm
  quantise     x (M, K) to E4M3 codes, a scale for every 128 values of a row
               (and, for a training step, of a column)
  linear       act(x W^T + bias) with x quantised on the way and W in codes
               with a scale for every 128 x 128 block
  product      the same from codes that are there already
  linear_grad  dx, dW and dbias of the linear layer: dy in codes both ways

The codes of a BlockFp8 are (rows, 128 * blocks) bytes, zero past k, and its
scales (blocks, rows), or (blocks, row blocks) for a weight. The scale of a
block is its largest magnitude over 448, or 1 where that magnitude is below
448 * 2**-126; a code is the E4M3 byte nearest x * (1 / scale), ties to even,
below 2**-6 at most 7 * 2**-9 as the codec of this framework has it.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
EPS = 1e-5


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # One token through a norm of an ordinary width: the smallest call, all latency.
        dict(name="norm_token", kind="norm", M=1, D=1024, dtype="bfloat16"),
        # The token mixer's norm at its serving size, 8 x 4096 tokens, d = 256, fp32 as this framework keeps activations.
        dict(name="norm_mixer", kind="norm", M=32768, D=256, dtype="float32"),
        # A wide norm ahead of an FP8 product, a prefill or training step of 16384 tokens.
        dict(name="norm_fp8_wide", kind="norm_fp8", M=16384, D=4096, dtype="bfloat16"),
        # Its backward pass; the weight's gradient sums 16384 rows.
        dict(name="norm_grad_wide", kind="norm_grad", M=16384, D=4096, dtype="bfloat16"),
        # A ragged backward pass: an odd number of rows of a width that no vector length divides.
        dict(name="norm_grad_ragged", kind="norm_grad", M=12289, D=1001, dtype="float32"),
        # What a training step makes of an activation: codes along both axes from one read.
        dict(name="quantise_both", kind="quantise", M=16384, K=4096, dtype="bfloat16", columns=True),
        # Rows alone, of an odd width whose last block is part of one: a serving batch.
        dict(name="quantise_ragged", kind="quantise", M=1537, K=2021, dtype="float32", columns=False),
        # One new token through a square layer: reads the weight once.
        dict(name="linear_token", kind="linear", M=1, K=4096, N=4096, dtype="bfloat16", act="none", bias=False),
        # The token mixer's qkv projection, 8 x 4096 tokens, 256 -> 768, fp32 in and out.
        dict(name="linear_mixer", kind="linear", M=32768, K=256, N=768, dtype="float32", act="none", bias=True),
        # A large product of codes, as a prefill runs it after norm_fp8. The largest.
        dict(name="product_large", kind="product", M=8192, K=8192, N=8192, dtype="bfloat16", act="none", bias=False),
        # The operator network's trunk layer trained: 65536 query points, 1024 -> 1024.
        dict(name="linear_grad_trunk", kind="linear_grad", M=65536, K=1024, N=1024, dtype="bfloat16"),
        # A ragged training step: no size a multiple of a tile or a block.
        dict(name="linear_grad_ragged", kind="linear_grad", M=5003, K=1000, N=1544, dtype="float32"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature width: mostly a multiple of 128 or 8, sometimes any number."""
    v = _logint(rng, lo, hi)
    step = rng.choice((128, 128, 8, 1))
    return max(lo, v // step * step)


def draw(rng):
    kind = rng.choice(("norm", "norm_fp8", "norm_grad", "quantise", "linear", "linear", "product", "linear_grad"))
    dtype = rng.choice(sorted(DTYPES))
    if kind in ("norm", "norm_fp8", "norm_grad"):
        D = _width(rng, 64, 16384)
        M = _logint(rng, 1, max(2, min(131072, 16384 * 4096 // D)))
        return dict(kind=kind, M=M, D=D, dtype=dtype)
    if kind == "quantise":
        K = _width(rng, 64, 16384)
        M = _logint(rng, 1, max(2, min(131072, 16384 * 4096 // K)))
        return dict(kind=kind, M=M, K=K, dtype=dtype, columns=rng.random() < 0.5)
    K, N = _width(rng, 64, 8192), _width(rng, 64, 8192)
    M = _logint(rng, 1, max(2, min(65536, 65536 * 1024 * 1024 // (K * N))))
    if kind == "linear_grad":
        return dict(kind=kind, M=M, K=K, N=N, dtype=dtype)
    return dict(kind=kind, M=M, K=K, N=N, dtype=dtype, act=rng.choice(("none", "relu", "gelu")), bias=rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------

def _blocks(n):
    return -(-n // 128)


def _activation(g, M, K, dtype):
    """Activations of a residual stream: normal values, each row with a level of
    its own, one feature in 64 some times larger."""
    x = torch.randn(M, K, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(M, 1, generator=g, device=DEV))
    x *= 1 + 7 * (torch.rand(K, generator=g, device=DEV) < 1 / 64).float()
    return x.to(DTYPES[dtype])


def _weight_blob(W):
    """Codes (N, 128 * blocks) and scales (blocks, row blocks) of 128 x 128 blocks."""
    N, K = W.shape
    nb, kb = _blocks(N), _blocks(K)
    P = torch.zeros(nb * 128, kb * 128, device=DEV)
    P[:N, :K] = W
    P = P.view(nb, 128, kb, 128)
    s = P.abs().amax(dim=(1, 3)) / 448
    q = _round_e4m3(P / s[:, None, :, None])
    codes = q.reshape(nb * 128, kb * 128)[:N].contiguous().to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), s.t().contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    s = dict(case)
    if kind in ("norm", "norm_fp8", "norm_grad"):
        M, D = case["M"], case["D"]
        s["x"] = _activation(g, M, D, case["dtype"])
        s["weight"] = 1 + 0.1 * torch.randn(D, generator=g, device=DEV)
        s["bias"] = 0.1 * torch.randn(D, generator=g, device=DEV)
        if kind == "norm_grad":
            s["dy"] = (torch.randn(M, D, generator=g, device=DEV) / math.sqrt(D)).to(dtype)
            v = s["x"].double()
            s["mean"] = v.mean(1).float()
            s["rstd"] = (v.var(1, unbiased=False) + EPS).rsqrt().float()
        return s
    if kind == "quantise":
        s["x"] = _activation(g, case["M"], case["K"], case["dtype"])
        return s
    M, K, N = case["M"], case["K"], case["N"]
    W = (2 * torch.rand(N, K, generator=g, device=DEV) - 1) / math.sqrt(K)
    x = _activation(g, M, K, case["dtype"])
    if kind == "linear_grad":
        # What the forward pass kept: x in codes along its columns, and the weight's codes transposed.
        s["x_codes"], s["x_scales"] = _quantise(x.t())
        w_codes, w_scales = _weight_blob(W)
        kb, nb = w_scales.shape
        t = torch.zeros(K, nb * 128, dtype=torch.uint8, device=DEV)
        t[:, :N] = w_codes[:, :K].t()
        s["w_codes"], s["w_scales"] = t, w_scales.t().contiguous()
        s["dy"] = (torch.randn(M, N, generator=g, device=DEV) / math.sqrt(M * N)).to(dtype)
        return s
    s["w_codes"], s["w_scales"] = _weight_blob(W)
    s["b"] = 0.1 * torch.randn(N, generator=g, device=DEV) if case["bias"] else None
    if kind == "product":
        s["x_codes"], s["x_scales"] = _quantise(x)
    else:
        s["x"] = x
    return s


# ---- the plain form --------------------------------------------------------------

def _round_e4m3(v):
    """The E4M3 value of |v| <= 448 after the codec's cap below 2**-6."""
    v = torch.where(v.abs() < 2.0 ** -6, v.clamp(-7 * 2.0 ** -9, 7 * 2.0 ** -9), v.clamp(-448, 448))
    return v.to(torch.float8_e4m3fn).float()


def _quantise(x):
    """Codes (M, 128 * blocks) and scales (blocks, M) of the rows of x."""
    M, K = x.shape
    kb = _blocks(K)
    P = torch.zeros(M, kb * 128, device=x.device)
    P[:, :K] = x
    P = P.view(M, kb, 128)
    amax = P.abs().amax(2)
    # Divided by a tensor: by a number torch multiplies with its rounded inverse instead.
    s = torch.where(amax < 448 * 2.0 ** -126, torch.ones_like(amax), amax / torch.full_like(amax, 448))
    q = _round_e4m3(P * (torch.ones_like(s) / s)[:, :, None])
    return q.view(M, kb * 128).to(torch.float8_e4m3fn).view(torch.uint8), s.t().contiguous()


def _values(codes, scales):
    """The numbers that codes (R, 128 * blocks) with scales (blocks, R or row blocks) stand for."""
    R = codes.shape[0]
    v = codes.view(torch.float8_e4m3fn).float().view(R, -1, 128)
    s = scales.t()
    if s.shape[0] != R:
        s = s.repeat_interleave(128, 0)[:R]
    return (v * s[:, :, None]).view(R, -1)


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain(s):
    kind, dtype = s["kind"], DTYPES[s["dtype"]]
    if kind in ("norm", "norm_fp8"):
        x = s["x"].float()
        mean = x.mean(1)
        c = x - mean[:, None]
        rstd = 1 / torch.sqrt((c * c).mean(1) + EPS)
        y = c * rstd[:, None] * s["weight"] + s["bias"]
        if kind == "norm":
            return y.to(dtype), mean, rstd
        codes, scales = _quantise(y)
        return codes.view(torch.float8_e4m3fn), scales, mean, rstd
    if kind == "norm_grad":
        dy, xh = s["dy"].float(), (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * s["weight"]
        dx = s["rstd"][:, None] * (g - g.mean(1)[:, None] - xh * (g * xh).mean(1)[:, None])
        return dx.to(dtype), (dy * xh).sum(0), dy.sum(0)
    if kind == "quantise":
        x = s["x"].float()
        out = [_quantise(x)] + ([_quantise(x.t())] if s["columns"] else [])
        return [t for codes, scales in out for t in (codes.view(torch.float8_e4m3fn), scales)]
    if kind == "linear_grad":
        dy = s["dy"].float()
        rows, cols = _quantise(dy), _quantise(dy.t())
        dx = _values(*rows) @ _values(s["w_codes"], s["w_scales"]).t()
        dw = _values(*cols) @ _values(s["x_codes"], s["x_scales"]).t()
        return dx.to(dtype), dw, dy.sum(0)
    xc, xs = (s["x_codes"], s["x_scales"]) if kind == "product" else _quantise(s["x"].float())
    z = _values(xc, xs) @ _values(s["w_codes"], s["w_scales"]).t()
    if s["b"] is not None:
        z = z + s["b"]
    return _act(z, s["act"]).to(dtype)


# ---- the framework's operators ------------------------------------------------------

def _framework(s):
    from neuroflow_amd import block_fp8 as B
    from neuroflow_amd import norm as L

    kind = s["kind"]
    if kind == "norm":
        return L.layer_norm(s["x"], s["weight"], s["bias"], EPS, return_stats=True)
    if kind == "norm_fp8":
        q, mean, rstd = L.layer_norm_fp8(s["x"], s["weight"], s["bias"], EPS, return_stats=True)
        return q.codes.view(torch.float8_e4m3fn), q.scales, mean, rstd
    if kind == "norm_grad":
        return L.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
    if kind == "quantise":
        out = B.quantise_both(s["x"]) if s["columns"] else [B.quantise(s["x"])]
        return [t for q in out for t in (q.codes.view(torch.float8_e4m3fn), q.scales)]
    if kind == "linear_grad":
        x_cols = B.BlockFp8(s["x_codes"], s["x_scales"], s["M"])
        w_t = B.BlockFp8(s["w_codes"], s["w_scales"], s["N"])
        return B.linear_backward(s["dy"], x_cols, w_t)
    w = B.BlockFp8(s["w_codes"], s["w_scales"], s["K"])
    if kind == "product":
        x = B.BlockFp8(s["x_codes"], s["x_scales"], s["K"])
        return B.matmul(x, w, s["b"], s["act"], DTYPES[s["dtype"]])
    return B.linear(s["x"], w, s["b"], s["act"])


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    kind, M = case["kind"], case["M"]
    e = 2 if case["dtype"] == "bfloat16" else 4
    if kind in ("norm", "norm_fp8", "norm_grad"):
        D = case["D"]
        if kind == "norm":
            return {"bytes": 2 * e * M * D + 8 * D + 8 * M, "flops": 8 * M * D}
        if kind == "norm_fp8":
            return {"bytes": (e + 1) * M * D + 4 * M * _blocks(D) + 8 * D + 8 * M, "flops": 11 * M * D}
        return {"bytes": 3 * e * M * D + 12 * D + 8 * M, "flops": 14 * M * D}
    K = case["K"]
    if kind == "quantise":
        rows, cols = M * K + 4 * M * _blocks(K), M * K + 4 * K * _blocks(M)
        return {"bytes": e * M * K + rows + (cols if case["columns"] else 0), "flops": (6 if case["columns"] else 3) * M * K}
    N = case["N"]
    weight = N * K + 4 * _blocks(N) * _blocks(K)
    if kind == "linear_grad":
        x = M * K + 4 * K * _blocks(M)
        return {"bytes": e * M * N + x + weight + e * M * K + 4 * N * K + 4 * N, "flops": 4 * M * N * K}
    x = M * K + 4 * M * _blocks(K) if kind == "product" else e * M * K
    return {"bytes": x + weight + (4 * N if case["bias"] else 0) + e * M * N, "flops": 2 * M * N * K}


# ---- the definition in 64 bits --------------------------------------------------------------

def _nearest64(v):
    """The E4M3 value nearest v, ties to even, by its exponent; the cap below 2**-6 as above."""
    a = v.abs().clamp(max=448)
    e = torch.frexp(a)[1].clamp(min=-5) - 1
    step = torch.ldexp(torch.ones_like(a), e - 3)
    q = torch.round(a / step) * step
    q = torch.where(a < 2.0 ** -6, q.clamp(max=7 * 2.0 ** -9), q)
    return torch.where(v < 0, -q, q)


def _quantise64(x):
    """Code values (M, blocks, 128) and scales (M, blocks) of x (M, K)."""
    M, K = x.shape
    P = torch.nn.functional.pad(x.double(), (0, -K % 128)).view(M, -1, 128)
    top = P.abs().max(2).values
    s = torch.where(top < 448 * 2.0 ** -126, torch.ones_like(top), top / 448)
    return _nearest64(P / s[:, :, None]), s


def _decode64(codes, scales, block):
    """Code bytes by sign, exponent and mantissa, times the scale of their block."""
    c = codes.int()
    e, m = (c >> 3) & 15, (c & 7).double()
    a = torch.where(e == 0, m * 2.0 ** -9, torch.ldexp(1 + m / 8, e - 7))
    v = torch.where(c >= 128, -a, a)
    at = torch.arange(codes.shape[0], device=codes.device) // block
    return v * scales.double()[:, at].t().repeat_interleave(128, 1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind in ("norm", "norm_fp8"):
        x = s["x"].double()
        mean, var = x.mean(1), x.var(1, unbiased=False)
        rstd = (var + EPS) ** -0.5
        y = (x - mean[:, None]) * (rstd[:, None] * s["weight"].double()) + s["bias"].double()
        if kind == "norm":
            return y, mean, rstd
        # No code of its own: where y lies between two codes, its last bits in 32 decide.
        return None, _quantise64(y)[1].t(), mean, rstd
    if kind == "norm_grad":
        # dx = W J with J the Jacobian of (x - mean) * rstd, applied to weight * dy.
        x, dy = s["x"].double(), s["dy"].double()
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
        h = (x - mean) * rstd
        g = dy * s["weight"].double()
        D = x.shape[1]
        dx = rstd / D * (D * g - g.sum(1, keepdim=True) - h * (g * h).sum(1, keepdim=True))
        return dx, (dy * h).sum(0), dy.sum(0)
    if kind == "quantise":
        out = []
        for x in (s["x"], s["x"].t())[:2 if s["columns"] else 1]:
            q, sc = _quantise64(x)
            out += [q.flatten(1), sc.t()]
        return out
    if kind == "linear_grad":
        dy = s["dy"].double()
        rows, rs = _quantise64(dy)
        dx = (rows * rs[:, :, None]).flatten(1) @ _decode64(s["w_codes"], s["w_scales"], 128).t()
        del rows
        cols, cs = _quantise64(dy.t())
        dw = (cols * cs[:, :, None]).flatten(1) @ _decode64(s["x_codes"], s["x_scales"], 1).t()
        return dx, dw, dy.sum(0)
    if kind == "product":
        x = _decode64(s["x_codes"], s["x_scales"], 1)
    else:
        q, sc = _quantise64(s["x"])
        x = (q * sc[:, :, None]).flatten(1)
    z = x @ _decode64(s["w_codes"], s["w_scales"], 128).t()
    if s["b"] is not None:
        z = z + s["b"].double()
    if s["act"] == "relu":
        return torch.maximum(z, torch.zeros_like(z))
    if s["act"] == "gelu":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z
