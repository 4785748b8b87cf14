"""The global norm of gradients and their clipping against 64 bits: sizes around
a chunk, alignments, mixed types, many tensors, infinities, graphs."""
import math

import pytest
import torch

from neuroflow_amd import _lib, grads
from residual_reference import U, gen, half, within

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
CHUNK = 8192


def make(sizes, seed, types=(F32,), offset=0):
    """Tensors of the sizes, their types in turn, each `offset` elements into its buffer."""
    g = gen(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = types[i % len(types)]
        buf = torch.full((n + offset + 9,), float("nan"), device="cuda", dtype=dt)
        v = buf[offset:offset + n]
        v.copy_(torch.randn(n, generator=g, device="cuda") * math.exp((i % 7) - 3))
        out.append(v)
    return out


def norm64(ts):
    return float(sum(t.double().square().sum() for t in ts)) ** 0.5


def check_clip(ts, max_norm, outs, norm):
    want = norm64(ts)
    assert norm.dtype == F32 and norm.shape == () and abs(float(norm) - want) <= 1.01 * U * want
    c = 1.0 if want <= max_norm else max_norm / want
    for t, o in zip(ts, outs):
        exact = t.double() * c
        # The factor's rounding, the product's, the result's; below the type's
        # smallest normal a rounding is half of its smallest step.
        within(o, exact, exact.abs() * (2 * U + half(o.dtype)) * 1.01 + 2.0 ** -133)


SETS = [[1], [7], [8], [CHUNK - 1], [CHUNK], [CHUNK + 1], [3 * CHUNK + 5, 1, 2], [0, 5, 0, 0, 100, 0], [1] * 130,
        [17] * 119 + [CHUNK + 3], [300] * 121, [2 * CHUNK] * 300, [5_000_000, 3, 1_000_001]]


@pytest.mark.parametrize("types", [(F32,), (BF16,), (BF16, F32)], ids=["f32", "bf16", "mixed"])
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip(gpu, sizes, types):
    for offset in (0, 1, 3):
        ts = make(sizes, len(sizes), types, offset)
        want = norm64(ts)
        n = grads.global_norm(ts)
        assert abs(float(n) - want) <= 1.01 * U * want
        outs = [torch.empty_like(t) for t in ts]
        check_clip(ts, want / 3, outs, grads.clip_by_global_norm(ts, want / 3, out=outs))
        check_clip(ts, want * 2, outs, grads.clip_by_global_norm(ts, want * 2, out=outs))
        assert all(torch.equal(a, b) for a, b in zip(ts, outs))
        before = [t.clone() for t in ts]
        norm = grads.clip_by_global_norm(ts, want * 2)             # nothing to clip: left as they are
        assert float(norm) == float(n) and all(torch.equal(a, b) for a, b in zip(ts, before))
        versions = [t._version for t in ts]
        norm = grads.clip_by_global_norm(ts, want / 3)
        check_clip(before, want / 3, ts, norm)
        assert all(t._version > v for t, v in zip(ts, versions))


def test_surroundings_are_left(gpu):
    buf = torch.full((3 * CHUNK,), 7.0, device="cuda")
    ts = [buf[5:CHUNK + 6], buf[CHUNK + 6:CHUNK + 6 + 11], buf[2 * CHUNK + 1:2 * CHUNK + 2]]
    grads.clip_by_global_norm(ts, 1.0)
    assert bool((buf[:5] == 7).all()) and bool((buf[CHUNK + 17:2 * CHUNK + 1] == 7).all()) and bool((buf[2 * CHUNK + 2:] == 7).all())
    assert abs(norm64(ts) - 1) < 1e-5


def test_range(gpu):
    """Squares past fp32's range either way, and values of both ends together."""
    for scale in (1e30, 1e-30, 1e-42):
        ts = [torch.full((1000,), scale, device="cuda"), torch.full((9,), -scale, device="cuda")]
        want = norm64(ts)
        assert abs(float(grads.global_norm(ts)) - want) <= 1.01 * U * want + 2.0 ** -150
    ts = [torch.tensor([3e38, 3e38], device="cuda")]
    assert math.isinf(float(grads.global_norm(ts)))               # 4.2e38 does not fit fp32
    outs = [torch.empty(2, device="cuda")]
    grads.clip_by_global_norm(ts, 1.0, out=outs)
    # The factor, 2.4e-39, is a subnormal: half its step is 3e-7 of it.
    within(outs[0], torch.full((2,), 0.5 ** 0.5, device="cuda", dtype=torch.float64), 5 * U)


def test_special_values(gpu):
    for bad, norm_is in ((float("nan"), math.isnan), (float("inf"), math.isinf)):
        ts = make([1000, 20], 3, (F32, BF16))
        ts[1][3] = bad
        norm = grads.clip_by_global_norm(ts, 1.0)
        assert norm_is(float(norm))
        if math.isnan(bad):
            assert bool(torch.isnan(ts[0]).all()) and bool(torch.isnan(ts[1]).all())
        else:
            assert not bool(ts[0].any()) and bool(torch.isnan(ts[1][3])) and int(ts[1].isnan().sum()) == 1
    ts = [torch.zeros(100, device="cuda"), torch.zeros(0, device="cuda")]
    assert float(grads.clip_by_global_norm(ts, 1.0)) == 0 and not bool(ts[0].any())
    assert float(grads.clip_by_global_norm(ts, 0.0)) == 0
    ts = make([100], 4)
    grads.clip_by_global_norm(ts, 0.0)
    assert not bool(ts[0].any())
    assert float(grads.global_norm([torch.zeros(0, device="cuda")])) == 0


def test_same_bits_and_graph(gpu):
    ts = make([100_000, 777, 50_000], 5, (BF16, F32))
    outs = [torch.empty_like(t) for t in ts]
    def step():
        return grads.clip_by_global_norm(ts, 1.0, out=outs), *outs
    first = [t.clone() for t in step()]
    assert all(torch.equal(a, b) for a, b in zip(step(), first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (6, 7, 8):
        for t, v in zip(ts, make([100_000, 777, 50_000], seed, (BF16, F32))):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(step(), got))
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        again = [t.clone() for t in step()]
        torch.cuda.current_stream().synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, got))


def test_refusals(gpu):
    t = torch.ones(100, device="cuda")
    for bad in (lambda: grads.global_norm([t.half()]), lambda: grads.global_norm([t.cpu()]), lambda: grads.global_norm([None]),
                lambda: grads.clip_by_global_norm([t], 1.0, out=[t.cpu()])):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: grads.global_norm([]), lambda: grads.global_norm([t[::2]]),
                lambda: grads.clip_by_global_norm([t], 1.0, out=[]), lambda: grads.clip_by_global_norm([t], 1.0, out=[t[:50]]),
                lambda: grads.clip_by_global_norm([t], 1.0, out=[t.bfloat16()]),
                lambda: grads.clip_by_global_norm([t.clone().requires_grad_()], 1.0)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: grads.clip_by_global_norm([t], -1.0), lambda: grads.clip_by_global_norm([t], float("nan")),
                lambda: grads.clip_by_global_norm([t, t], 1.0), lambda: grads.clip_by_global_norm([t[:60], t[50:]], 1.0),
                lambda: grads.clip_by_global_norm([t[:50], t[50:]], 1.0, out=[t[50:], t[:50]]),
                lambda: grads.clip_by_global_norm([t[:50]], 1.0, out=[t[1:51]])):
        with pytest.raises(_lib.NflowError):
            bad()
    assert bool((t == 1).all())
    grads.global_norm([t, t])                                     # reading one twice is fine
    grads.clip_by_global_norm([t[:50], t[50:]], 1.0)
