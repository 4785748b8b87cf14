"""A norm and a block-FP8 projection, trained and then served.

The layer is what stands at the head of a token mixer block: layer norm over
the features, then a projection (256 -> 768 by default, the mixer's qkv), with
its weight in 128 x 128 blocks of E4M3 codes and its input quantised in 1 x 128
blocks. The master weight is fp32; every step quantises it, runs the forward
and backward pass in FP8 and takes a step of plain gradient descent towards a
teacher of the same form. Then the trained layer answers single tokens.

    python examples/norm_fp8_layer.py [--steps 60] [--tokens 8192] [--dtype bf16]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from neuroflow_amd import block_fp8, norm


class NormProjection:
    """norm -> block-FP8 linear: fp32 parameters, explicit forward and backward."""

    def __init__(self, d_in: int, d_out: int, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.gamma = torch.ones(d_in, device="cuda")
        self.beta = torch.zeros(d_in, device="cuda")
        self.W = (2 * torch.rand(d_out, d_in, generator=g, device="cuda") - 1) / d_in ** 0.5
        self.bias = torch.zeros(d_out, device="cuda")

    def forward(self, x: torch.Tensor):
        """y, and what the backward pass needs."""
        h, mean, rstd = norm.layer_norm(x, self.gamma, self.beta, return_stats=True)
        h_rows, h_columns = block_fp8.quantise_both(h)
        w, w_t = block_fp8.quantise_weight(self.W, transposed=True)
        y = block_fp8.matmul(h_rows, w, self.bias, out_dtype=x.dtype)
        return y, (x, mean, rstd, h_columns, w_t)

    def backward(self, dy: torch.Tensor, kept):
        """dx, and the parameters' gradients in the order of parameters()."""
        x, mean, rstd, h_columns, w_t = kept
        dh, dW, dbias = block_fp8.linear_backward(dy, h_columns, w_t)
        dx, dgamma, dbeta = norm.layer_norm_backward(dh, x, self.gamma, mean, rstd)
        return dx, (dgamma, dbeta, dW, dbias)

    def parameters(self):
        return self.gamma, self.beta, self.W, self.bias


class ServedProjection:
    """The trained layer for inference: the weight's codes laid out once."""

    def __init__(self, layer: NormProjection):
        self.gamma, self.beta, self.bias = layer.gamma, layer.beta, layer.bias
        self.w = block_fp8.quantise_weight(layer.W)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[0] == 1:     # one token: the projection quantises its input in the same launch
            return block_fp8.linear(norm.layer_norm(x, self.gamma, self.beta), self.w, self.bias)
        q = norm.layer_norm_fp8(x, self.gamma, self.beta)
        return block_fp8.matmul(q, self.w, self.bias, out_dtype=x.dtype)


def train(steps: int = 60, tokens: int = 8192, d_in: int = 256, d_out: int = 768, dtype=torch.bfloat16,
          rate: float = 0.2):
    """(losses, trained layer): mean squared error to a teacher's outputs."""
    g = torch.Generator(device="cuda").manual_seed(1)
    teacher, layer = NormProjection(d_in, d_out, 2), NormProjection(d_in, d_out, 3)
    teacher.gamma += 0.2 * torch.randn(d_in, generator=g, device="cuda")
    teacher.bias += 0.2 * torch.randn(d_out, generator=g, device="cuda")
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, d_in, generator=g, device="cuda").to(dtype)
        want, _ = teacher.forward(x)
        y, kept = layer.forward(x)
        diff = y.float() - want.float()
        losses.append((diff * diff).mean())
        _, grads = layer.backward((diff * (2 / tokens)).to(dtype), kept)
        for p, d in zip(layer.parameters(), grads):
            p.sub_(d, alpha=rate)
    return [float(v) for v in losses], layer


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=8192)
    ap.add_argument("--dtype", choices=("fp32", "bf16"), default="bf16")
    a = ap.parse_args()
    dtype = torch.float32 if a.dtype == "fp32" else torch.bfloat16
    losses, layer = train(a.steps, a.tokens, dtype=dtype)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.5f} in {a.steps} steps")
    served = ServedProjection(layer)
    x = torch.randn(4, 256, device="cuda").to(dtype)
    batch, single = served(x), torch.cat([served(x[i:i + 1]) for i in range(4)])
    print(f"4 tokens at once and one by one differ by at most {float((batch - single).abs().max()):.2e}")


if __name__ == "__main__":
    main()
