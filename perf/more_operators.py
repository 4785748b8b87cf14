"""A residual block's unquantised side, as measurable cases: RMS norm with the
residual's addition, the linear layer with its epilogue, gradient clipping.

Around the 8-bit products of a transformer or token-mixer block stand a norm
that takes the residual stream in, the layers that stay in bf16 or fp32, and,
when the block trains, the clipping of its gradients.  Each case here is one
call of that path, through neuroflow_amd.norm, neuroflow_amd.dense and
neuroflow_amd.grads:

  rms          t = x + residual, y = t * rstd * weight with rstd =
               1 / sqrt(mean(t^2) + eps) over the last axis of t (M, D); y, t, rstd
  rms_fp8      the same, y as E4M3 codes with a scale for every 128 features
  rms_grad     dt (with the gradient that t has from its other use) and dweight
  linear       y = act(z), z = x W^T + bias + residual; z too where it is kept
               for the backward pass
  linear_grad  dz = dy act'(z); dx = dz W, dW = dz^T x, dbias = the sum of dz's rows
  clip         norm = the root of the sum of squares over all gradients; each
               gradient times min(1, max_norm / norm)
  norm         that norm alone

t's norm is of the sum before its rounding to x's type.  The gradient dz that
the products of linear_grad take is the one it returns, in x's type; the plain
form keeps it in 32 bits until its end.  Codes and scales are those of
neuroflow_amd.block_fp8: the scale of a block is its largest magnitude over
448, or 1 where that magnitude is below 448 * 2**-126; a code is the E4M3 byte
nearest y * (1 / scale), ties to even, below 2**-6 at most 7 * 2**-9.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
EPS = 1e-5
GELU = math.sqrt(2 / math.pi), 0.044715


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # One token's step into a block: the stream takes the last layer's output and is normed. All latency.
        dict(name="rms_token", kind="rms", M=1, D=1024, dtype="bfloat16", residual=True),
        # The same at the token mixer's serving size, 8 x 4096 tokens, d = 256, fp32 as this framework keeps activations.
        dict(name="rms_mixer", kind="rms", M=32768, D=256, dtype="float32", residual=True),
        # Ahead of an FP8 product, a prefill or training step of 16384 tokens in a wide model.
        dict(name="rms_fp8_wide", kind="rms_fp8", M=16384, D=4096, dtype="bfloat16", residual=True),
        # Its backward pass, the residual stream's own gradient joined on the way.
        dict(name="rms_grad_wide", kind="rms_grad", M=16384, D=4096, dtype="bfloat16", residual=True),
        # One new token through a layer kept in bf16, added to the stream: reads the weight once.
        dict(name="linear_token", kind="linear", M=1, K=4096, N=4096, dtype="bfloat16", act="none", bias=False, residual=True, pre=False),
        # The token mixer's output projection onto its stream, 8 x 4096 tokens, 256 -> 256, in fp32.
        dict(name="linear_mixer", kind="linear", M=32768, K=256, N=256, dtype="float32", act="none", bias=True, residual=True, pre=False),
        # A ragged batch: no size a multiple of a tile, rows of odd length in memory.
        dict(name="linear_ragged", kind="linear", M=1537, K=2021, N=1001, dtype="bfloat16", act="gelu", bias=True, residual=True, pre=True),
        # The largest product, a layer of a wide model over a long prefill.
        dict(name="linear_large", kind="linear", M=8192, K=8192, N=8192, dtype="bfloat16", act="gelu", bias=True, residual=False, pre=False),
        # The operator network's trunk layer trained in bf16: 65536 query points, 1024 -> 1024, GELU.
        dict(name="linear_grad_trunk", kind="linear_grad", M=65536, K=1024, N=1024, dtype="bfloat16", act="gelu"),
        # A ragged training step in fp32.
        dict(name="linear_grad_ragged", kind="linear_grad", M=5003, K=1000, N=1544, dtype="float32", act="none"),
        # The token mixer's gradients, 6 blocks of d = 256: many small tensors, most of them a few KB.
        dict(name="clip_mixer", kind="clip", layers=6, d=256, dtype="float32", over=True, packed=False),
        # A wide model's share of gradients on one GPU, weights in bf16 and norms in fp32: from HBM.
        dict(name="clip_wide", kind="clip", layers=10, d=4096, dtype="mixed", over=True, packed=False),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature width: mostly a multiple of 128 or 8, sometimes any number."""
    v = _logint(rng, lo, hi)
    step = rng.choice((128, 128, 8, 1))
    return max(lo, v // step * step)


def draw(rng):
    kind = rng.choice(("rms", "rms_fp8", "rms_grad", "linear", "linear", "linear", "linear_grad", "linear_grad", "clip", "norm"))
    if kind in ("clip", "norm"):
        case = dict(kind=kind, layers=rng.randint(1, 10), d=_width(rng, 64, 4096), dtype=rng.choice(("float32", "bfloat16", "mixed")),
                    packed=rng.random() < 0.5)
        if case["d"] > 2048 and case["dtype"] == "float32":
            case["layers"] = min(case["layers"], 5)
        return dict(case, over=rng.random() < 0.7) if kind == "clip" else case
    dtype = rng.choice(sorted(DTYPES))
    if kind in ("rms", "rms_fp8", "rms_grad"):
        D = _width(rng, 64, 16384)
        M = _logint(rng, 1, max(2, min(131072, 16384 * 4096 // D)))
        return dict(kind=kind, M=M, D=D, dtype=dtype, residual=rng.random() < 0.7)
    most = 65536 * 1024 * 1024 if dtype == "bfloat16" else 65536 * 1024 * 256
    K, N = _width(rng, 64, 8192), _width(rng, 64, 8192)
    M = _logint(rng, 1, max(2, min(65536, most // (K * N))))
    act = rng.choice(("none", "relu", "gelu"))
    if kind == "linear_grad":
        return dict(kind=kind, M=M, K=K, N=N, dtype=dtype, act=act)
    return dict(kind=kind, M=M, K=K, N=N, dtype=dtype, act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                pre=act != "none" and rng.random() < 0.5)


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


def _shapes(case):
    """A mixer block's parameters: norm, qkv projection, output projection; and their types."""
    d = case["d"]
    big = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    small = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32
    block = [((d,), small), ((d,), small), ((3 * d, d), big), ((3 * d,), small), ((d, d), big), ((d,), small)]
    return block * case["layers"]


def _gradients(g, case):
    """Gradients of a backward pass, each tensor with a level of its own; packed:
    views one after another into a buffer per type, an element off any alignment."""
    shapes = _shapes(case)
    level = 1.0 if case.get("over", True) else 1e-6
    flat = {}
    if case["packed"]:
        for dt in {dt for _, dt in shapes}:
            flat[dt] = [torch.empty(1 + sum(math.prod(s) for s, t in shapes if t == dt), dtype=dt, device=DEV), 1]
    out = []
    for shape, dt in shapes:
        v = torch.randn(shape, generator=g, device=DEV) * (level * 1e-2 * torch.exp(torch.randn((), generator=g, device=DEV)))
        if case["packed"]:
            buf, at = flat[dt]
            view = buf[at:at + v.numel()].view(shape)
            view.copy_(v)
            flat[dt][1] = at + v.numel()
            out.append(view)
        else:
            out.append(v.to(dt))
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    s = dict(case)
    if kind in ("clip", "norm"):
        s["grads"] = _gradients(g, case)
        if kind == "clip":
            s["max_norm"] = 1.0
            s["out"] = [torch.empty_like(t) for t in s["grads"]]
        return s
    dtype = DTYPES[case["dtype"]]
    M = case["M"]
    if kind in ("rms", "rms_fp8", "rms_grad"):
        D = case["D"]
        s["x"] = _activation(g, M, D, case["dtype"])
        s["weight"] = 1 + 0.1 * torch.randn(D, generator=g, device=DEV)
        s["r"] = _activation(g, M, D, case["dtype"]) if case["residual"] else None
        if kind == "rms_grad":
            s["dy"] = (torch.randn(M, D, generator=g, device=DEV) / math.sqrt(D)).to(dtype)
            s["rstd"] = (s["x"].double().square().mean(1) + EPS).rsqrt().float()
            if case["residual"]:
                s["r"] = (torch.randn(M, D, generator=g, device=DEV) / math.sqrt(D)).to(dtype)
        return s
    K, N = case["K"], case["N"]
    s["x"] = _activation(g, M, K, case["dtype"])
    s["W"] = ((2 * torch.rand(N, K, generator=g, device=DEV) - 1) / math.sqrt(K)).to(dtype)
    if kind == "linear_grad":
        s["dy"] = (torch.randn(M, N, generator=g, device=DEV) / math.sqrt(M * N)).to(dtype)
        s["z"] = torch.randn(M, N, generator=g, device=DEV).to(dtype) if case["act"] != "none" else None
        return s
    s["b"] = 0.1 * torch.randn(N, generator=g, device=DEV) if case["bias"] else None
    s["r"] = _activation(g, M, N, case["dtype"]) if case["residual"] else None
    return s


# ---- the plain form --------------------------------------------------------------

def _round_e4m3(v):
    """The E4M3 value of |v| <= 448 after the codec's cap below 2**-6."""
    v = torch.where(v.abs() < 2.0 ** -6, v.clamp(-7 * 2.0 ** -9, 7 * 2.0 ** -9), v.clamp(-448, 448))
    return v.to(torch.float8_e4m3fn)


def _quantise(y):
    """Codes (M, 128 * blocks) and scales (blocks, M) of the rows of y."""
    M, K = y.shape
    kb = _blocks(K)
    P = torch.zeros(M, kb * 128, device=y.device)
    P[:, :K] = y
    P = P.view(M, kb, 128)
    amax = P.abs().amax(2)
    # Divided by a tensor: by a number torch multiplies with its rounded inverse instead.
    s = torch.where(amax < 448 * 2.0 ** -126, torch.ones_like(amax), amax / torch.full_like(amax, 448))
    return _round_e4m3(P * (torch.ones_like(s) / s)[:, :, None]).view(M, kb * 128), s.t().contiguous()


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(GELU[0] * (z + GELU[1] * z * z * z)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    t = torch.tanh(GELU[0] * (z + GELU[1] * z * z * z))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * GELU[0] * (1 + 3 * GELU[1] * z * z)


def _global_norm(grads):
    return torch.sqrt(sum(t.double().square().sum() for t in grads))


def _plain(s):
    kind = s["kind"]
    if kind in ("clip", "norm"):
        norm = _global_norm(s["grads"])
        if kind == "norm":
            return norm.float()
        c = (s["max_norm"] / norm).clamp(max=1.0).float()
        for t, o in zip(s["grads"], s["out"]):
            o.copy_(t.float() * c)
        return norm.float(), s["out"]
    dtype = DTYPES[s["dtype"]]
    if kind in ("rms", "rms_fp8"):
        t = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
        rstd = 1 / torch.sqrt((t * t).mean(1) + EPS)
        y = t * rstd[:, None] * s["weight"]
        y = (y.to(dtype),) if kind == "rms" else _quantise(y)
        return (*y, rstd) if s["r"] is None else (*y, t.to(dtype), rstd)
    if kind == "rms_grad":
        dy, h = s["dy"].float(), s["x"].float() * s["rstd"][:, None]
        g = dy * s["weight"]
        dt = s["rstd"][:, None] * (g - h * (g * h).mean(1)[:, None])
        if s["r"] is not None:
            dt = dt + s["r"].float()
        return dt.to(dtype), (dy * h).sum(0)
    x, W = s["x"].float(), s["W"].float()
    if kind == "linear_grad":
        dz = s["dy"].float()
        if s["act"] != "none":
            dz = dz * _act_slope(s["z"].float(), s["act"])
        return (dz @ W).to(dtype), (dz.t() @ x).to(dtype), dz.sum(0), dz.to(dtype)
    z = x @ W.t()
    if s["b"] is not None:
        z = z + s["b"]
    if s["r"] is not None:
        z = z + s["r"].float()
    y = _act(z, s["act"]).to(dtype)
    return (y, z.to(dtype)) if s["pre"] else y


# ---- the framework's operators ------------------------------------------------------

def _framework(s):
    from neuroflow_amd import dense, grads
    from neuroflow_amd import norm as L

    kind = s["kind"]
    if kind == "norm":
        return grads.global_norm(s["grads"])
    if kind == "clip":
        return grads.clip_by_global_norm(s["grads"], s["max_norm"], out=s["out"]), s["out"]
    if kind == "rms":
        return L.rms_norm(s["x"], s["weight"], EPS, residual=s["r"], return_stats=True)
    if kind == "rms_fp8":
        q, *rest = L.rms_norm_fp8(s["x"], s["weight"], EPS, residual=s["r"], return_stats=True)
        return (q.codes.view(torch.float8_e4m3fn), q.scales, *rest)
    if kind == "rms_grad":
        return L.rms_norm_backward(s["dy"], s["x"], s["weight"], s["rstd"], dsum=s["r"])
    act = None if s["act"] == "none" else s["act"]
    if kind == "linear_grad":
        return dense.linear_backward(s["dy"], s["x"], s["W"], act, pre=s["z"])
    return dense.linear(s["x"], s["W"], s["b"], act, residual=s["r"], return_pre=s["pre"])


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("clip", "norm"):
        n = sum(math.prod(s) for s, _ in _shapes(case))
        e = sum(math.prod(s) * dt.itemsize for s, dt in _shapes(case))
        return {"bytes": (2 if kind == "clip" else 1) * e + 4, "flops": (3 if kind == "clip" else 2) * n}
    M = case["M"]
    e = 2 if case["dtype"] == "bfloat16" else 4
    if kind in ("rms", "rms_fp8", "rms_grad"):
        D, r = case["D"], 2 if case["residual"] else 0
        if kind == "rms":
            return {"bytes": (2 + r) * e * M * D + 4 * D + 4 * M, "flops": 5 * M * D}
        if kind == "rms_fp8":
            return {"bytes": ((1 + r) * e + 1) * M * D + 4 * M * _blocks(D) + 4 * D + 4 * M, "flops": 8 * M * D}
        return {"bytes": (3 + r // 2) * e * M * D + 8 * D + 4 * M, "flops": 10 * M * D}
    K, N = case["K"], case["N"]
    if kind == "linear_grad":
        z = 0 if case["act"] == "none" else e * M * N
        # dz is an output of its own where an activation makes it another tensor than dy.
        return {"bytes": e * (M * N + 2 * M * K + 2 * N * K) + 4 * N + 2 * z, "flops": 4 * M * N * K}
    rows = 1 + (1 if case["residual"] else 0) + (1 if case["pre"] else 0)
    return {"bytes": e * (M * K + N * K + rows * M * N) + (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}


# ---- the definition in 64 bits --------------------------------------------------------------

def _slope64(z, act):
    """act(z) and its derivative, the tanh GELU as z times a logistic function."""
    if act == "relu":
        return torch.maximum(z, torch.zeros_like(z)), torch.where(z > 0, 1.0, 0.0).double()
    if act == "none":
        return z, torch.ones_like(z)
    p = torch.sigmoid(2 * GELU[0] * (z + GELU[1] * z ** 3))
    return z * p, p + z * p * (1 - p) * 2 * GELU[0] * (1 + 3 * GELU[1] * z ** 2)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind in ("clip", "norm"):
        total = torch.zeros((), dtype=torch.float64, device=DEV)
        for t in s["grads"]:
            total += torch.linalg.vector_norm(t.double().flatten()) ** 2
        norm = total ** 0.5
        if kind == "norm":
            return norm
        c = min(1.0, s["max_norm"] / float(norm))
        return norm, [t.double() * c for t in s["grads"]]
    x = s["x"].double()
    if kind in ("rms", "rms_fp8"):
        t = x if s["r"] is None else x + s["r"].double()
        rstd = (torch.linalg.vector_norm(t, dim=1) ** 2 / t.shape[1] + EPS) ** -0.5
        y = t * (rstd[:, None] * s["weight"].double())
        if kind == "rms_fp8":
            # No code of its own: where y lies between two codes, its last bits in 32 decide.
            top = torch.nn.functional.pad(y, (0, -y.shape[1] % 128)).view(y.shape[0], -1, 128).abs().max(2).values
            y = (None, torch.where(top < 448 * 2.0 ** -126, torch.ones_like(top), top / 448).t())
        else:
            y = (y,)
        return (*y, rstd) if s["r"] is None else (*y, t, rstd)
    if kind == "rms_grad":
        # dt = J^T (weight * dy) with J the Jacobian of t * rstd.
        dy, rstd = s["dy"].double(), s["rstd"].double()[:, None]
        h = x * rstd
        g = dy * s["weight"].double()
        D = x.shape[1]
        dt = rstd / D * (D * g - h * (g * h).sum(1, keepdim=True))
        return dt if s["r"] is None else dt + s["r"].double(), (dy * h).sum(0)
    W = s["W"].double()
    if kind == "linear_grad":
        dz = s["dy"].double()
        if s["act"] != "none":
            dz = dz * _slope64(s["z"].double(), s["act"])[1]
        return dz @ W, dz.t() @ x, dz.sum(0), dz
    z = torch.nn.functional.linear(x, W)
    if s["b"] is not None:
        z += s["b"].double()
    if s["r"] is not None:
        z += s["r"].double()
    y = _slope64(z, s["act"])[0]
    return (y, z) if s["pre"] else y
