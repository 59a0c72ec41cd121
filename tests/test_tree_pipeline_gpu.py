"""Tree attention where a workgroup walks many tiles: the wide kernel's steps in
pairs with K two tiles ahead, the narrow kernels' stage that is refilled while the
other is read, with blocks of any size and blocks that are not there.

Tolerances as in test_tree_attention_gpu.py, with u = 2^-24, A the weighted mean
of |v|, d the largest scale * sum |q_d k_d|, T the attended rows:
  |out - exact| <= A (2 (D + 6) u d + (2 T + 8) u + w) + f + r |out| (1 + w)
  |lse - exact| <= (D + 6) u d + (T + 8) u + 4 u |lse|
w is half a step of the pool's type for the rounded weights (fp32: 0) and r half a
step of out's.  f: an fp16 weight below 2^-14 is off by at most half a step of the
subnormals, 2^-25, where the largest weight is at least 2^7: T 2^-32 max|v|."""
from __future__ import annotations

import random

import pytest
import torch

import tree_launch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def check(b, out, lse, exact, rows=slice(None)):
    ref, z, mean, dots = exact
    T, D = max(c + n for c, n in zip(b.lengths, b.nodes)), b.D
    w = 0.0 if b.dtype == F32 else HALF[b.dtype]
    tol = mean * (2 * (D + 6) * U * dots[..., None] + (2 * T + 8) * U + w) + HALF[b.dtype] * ref.abs() * (1 + w)
    if b.dtype == F16:
        tol = tol + T * 2.0 ** -32 * float(b.args["v_pool"].abs().max())
    off = (out[rows].double() - ref).abs() - tol
    assert bool(torch.isfinite(out[rows]).all()) and off.max().item() <= 0, f"off by {off.max().item():.3e} more than allowed"
    lt = (D + 6) * U * dots + (T + 8) * U + 4 * U * z.abs()
    assert bool(((lse[rows].double() - z).abs() <= lt).all())


def _lengths(seed, B, lo, hi):
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(B)]


@pytest.mark.parametrize("holes", [0.0, 0.06])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("H,nodes", [(8, 20), (8, 25), (8, 50), (28, 17), (8, 100), (40, 25)])
def test_wide_items_of_many_tiles(dev, H, nodes, dtype, D, holes):
    """Committed tiles in pairs, then the rest: of even and odd items, and of items that end in tree rows."""
    B = 16
    n = [nodes - i % 3 for i in range(B)]
    b = tree_launch.Batch(dev, lengths=_lengths(H + nodes, B, 2000, 8000), nodes=n, H=H, Hk=4, D=D, bs=16, dtype=dtype,
                          seed=nodes, holes=holes)
    c = b.cuts()
    assert c.shape.nw == {20: 2, 25: 2 if H == 8 else 8, 50: 4, 17: 4, 100: 8}[nodes] and c.L >= 6
    steps = [(min(t, tree - at) - 1) // 2 for at, t, tree in c.sizes]   # pairs of steps that an item takes
    assert max(steps) >= 2 and {t % 2 for (_, t, _), s in zip(c.sizes, steps) if s >= 2} == {0, 1}
    assert any(s >= 2 and at + t > tree for (at, t, tree), s in zip(c.sizes, steps))
    check(b, *b.run(), b.exact())


def test_wide_items_without_masks(dev):
    b = tree_launch.Batch(dev, lengths=_lengths(5, 12, 3000, 6000), nodes=[130 + i for i in range(12)], H=4, Hk=4, D=128, bs=24,
                          dtype=BF16, seed=5, masks=False)
    c = b.cuts()
    assert c.shape.nw == 8 and max(t for _, t, _ in c.sizes) > 6
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("holes", [0.0, 0.06])
@pytest.mark.parametrize("bs", [16, 24, 3])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_narrow_items_of_many_tiles(dev, dtype, D, bs, holes):
    """Three tiles a wave and more; the last ones of some items hold tree rows."""
    B = 34
    b = tree_launch.Batch(dev, lengths=_lengths(bs, B, 900, 2500), nodes=[1 + i % 8 for i in range(B)], H=32, Hk=8, D=D, bs=bs,
                          dtype=dtype, seed=bs, holes=holes)
    c = b.cuts()
    sizes = [t for _, t, _ in c.sizes]
    assert c.shape.nw == 1 and max(sizes) >= 24 and sum(t >= 12 for t in sizes) >= 20
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_narrow_items_of_few_units(dev, dtype, D):
    """One item a CU: one node of each request, as in a paged decode step."""
    b = tree_launch.Batch(dev, lengths=[12000, 7001, 9999, 8192], nodes=[1] * 4, H=32, Hk=8, D=D, bs=16, dtype=dtype, seed=D)
    c = b.cuts()
    assert c.shape.slots == 256 and max(t for _, t, _ in c.sizes) >= 12
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("nodes", [1, 12])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_small_weights_behind_a_large_one_are_not_lost(dev, dtype, nodes):
    """A first row of large score and no value, 2^-25.6 as much weight on each of the rows behind it."""
    B, T, H, Hk, D, bs = 80, 9000, 8 if nodes == 1 else 16, 4, 64, 16
    b = tree_launch.Batch(dev, lengths=[T] * B, nodes=[nodes] * B, H=H, Hk=Hk, D=D, bs=bs, dtype=dtype, seed=2, blocks=600,
                          masks=False)
    a = b.args
    a["q"].fill_(2.0 ** -3)
    a["k_pool"].zero_()
    a["v_pool"].fill_(1.0)
    a["block_table"].copy_(torch.arange(b.W, device=dev).expand(B, b.W))
    a["k_pool"][0, :, 0] = 17.75  # its score: 64 x 1/8 x 17.75 x 1/8, 25.6 log 2
    a["v_pool"][0, :, 0] = 0
    c = b.cuts()
    assert c.shape.nw == (1 if nodes == 1 or dtype == F32 else 2) and max(t for _, t, _ in c.sizes) * c.shape.kt > 5000
    check(b, *b.run(), b.exact(only=[0]), rows=slice(0, nodes))


@pytest.mark.parametrize("nodes", [3, 12])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("scale", [2.0 ** -5, 2.0 ** -3, 2.0 ** -2])
def test_huge_scores_stay_finite(dev, scale, dtype, nodes):
    """The largest exponents of a row are about 2^26, 2^28 and 2^29, where fp32's steps are 8, 32 and 64: out is a mean of
    V's rows all the same, in each channel between the least and the largest (a weight and out are off by half a step each)."""
    b = tree_launch.Batch(dev, lengths=[700, 3000], nodes=[nodes, nodes - 2], H=8, Hk=2, D=64, bs=16, dtype=dtype, seed=3, masks=False)
    for t in (b.args["q"], b.args["k_pool"]):
        t.mul_(2.0 ** 13).clamp_(-60000, 60000)
    b.args["v_pool"].abs_()
    out, lse = b.run(scale=scale)
    top = float(b.args["v_pool"].max()) * (1 + 2 * HALF[dtype]) * (1 + 8000 * U)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    assert float(lse.max()) > 2.0 ** 30 * scale
    assert float(out.min()) >= 0 and float(out.max()) <= top
