"""Rows rotated and written to a pool on the GPU, against the definition in
float64.

Tolerances, with u = 2^-24 and r half a step of the rows' type:
  norm      a sum of D squares, in any order (D + 1) u of it, its division by D,
            eps and the root: less than (D / 2 + 3) u of the quotient, which is
            multiplied twice: e = (D / 2 + 6) u of a channel
  rotation  two products and their difference: (|a c| + |b s|) (e + 3 u)
  rounding  r of the value; in fp16 below its normal range at most 2^-25"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import serving

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


class Case:
    def __init__(self, dev, *, N, H=8, Hk=2, D=64, R=None, bs=16, dtype=BF16, pairs=False, norm=True, norm32=False, far=500,
                 seed=0, eps=1e-6, long=True, lead=0):
        g = torch.Generator().manual_seed(seed)
        R = R or D
        self.D, self.dtype, self.pairs, self.eps, self.bs, self.dev = D, dtype, pairs, eps, bs, dev
        qkv = torch.randn(N, H + 2 * Hk, D + lead, generator=g).to(dtype).to(dev)[..., lead:]
        self.q, self.k, self.v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        angle = torch.arange(far, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2).double() / R)
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        self.pos = torch.randint(0, far, (N,), generator=g).to(torch.int64 if long else torch.int32).to(dev)
        P = -(-N // bs) + 3
        self.slots = torch.randperm(P * bs, generator=g)[:N].to(dev)
        w = lambda: (1 + 0.3 * torch.randn(D, generator=g)).to(F32 if norm32 else dtype).to(dev)  # noqa: E731
        self.qn, self.kn = (w(), w()) if norm else (None, None)
        self.kp, self.vp = (torch.randn(P, Hk, bs, D, generator=g).to(dtype).to(dev) for _ in range(2))

    def run(self, **kw):
        import halo_amd
        a = dict(q_norm=self.qn, k_norm=self.kn, eps=self.eps, interleaved=self.pairs)
        return halo_amd.rotate_rows(self.q, self.k, self.v, self.pos, self.cos, self.sin, self.slots, self.kp, self.vp,
                                    **{**a, **kw})

    def check(self, got=None):
        before = self.kp.clone(), self.vp.clone()
        got = self.run() if got is None else got
        P, Hk, bs, D = self.kp.shape
        cos, sin = (t[self.pos.long()].double().cpu().numpy() for t in (self.cos, self.sin))
        kept = (self.slots >= 0) & (self.slots < P * bs)
        at = self.slots[kept]
        rows = lambda t: t[at // bs, :, at % bs]  # noqa: E731
        for x, w, y, keep in ((self.q, self.qn, got, slice(None)), (self.k, self.kn, rows(self.kp), kept.cpu().numpy())):
            f = lambda t: t.double().cpu().numpy()  # noqa: E731
            ref, size = serving.rotate(f(x), None if w is None else f(w), self.eps, cos, sin, self.pairs)
            ref, size = ref[keep], size[keep]
            e = 0.0 if w is None else (D / 2 + 6) * U
            tol = size * (e + 3 * U) * (1 + HALF[self.dtype]) + HALF[self.dtype] * np.abs(ref)
            tol += 2.0 ** -25 if self.dtype == F16 else 0.0
            assert y.dtype == self.dtype and (np.abs(f(y) - ref) <= tol).all()
        assert torch.equal(rows(self.vp), self.v[kept])
        mask = torch.zeros(P * bs, dtype=torch.bool, device=self.dev)
        mask[at] = True
        mask = mask.view(P, 1, bs, 1).expand_as(self.kp)
        for now, was in zip((self.kp, self.vp), before):
            assert torch.equal(now[~mask], was[~mask])  # other rows as they were


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("N", [1, 2, 3, 33, 257])
def test_rows(dev, N, norm, pairs, D, dtype):
    Case(dev, N=N, D=D, dtype=dtype, pairs=pairs, norm=norm, seed=N).check()


@pytest.mark.parametrize("D,R", [(64, 16), (64, 32), (64, 48), (128, 16), (128, 80), (128, 112)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_parts_of_a_head(dev, D, R, pairs, dtype):
    Case(dev, N=19, D=D, R=R, dtype=dtype, pairs=pairs, seed=R).check()


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (28, 4), (32, 8), (8, 8), (40, 10), (128, 1)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N", [5, 1000])
def test_heads(dev, H, Hk, dtype, N):
    Case(dev, N=N, H=H, Hk=Hk, D=128, dtype=dtype, seed=H).check()


@pytest.mark.parametrize("bs", [1, 7, 24, 256])
def test_block_sizes(dev, bs):
    Case(dev, N=50, bs=bs, seed=bs).check()


def test_long_calls(dev):
    for dtype, N in ((BF16, 20000), (F16, 9001), (F32, 5003)):
        Case(dev, N=N, H=32, Hk=8, D=128, dtype=dtype, far=131072, seed=N).check()


def test_no_rows(dev):
    c = Case(dev, N=4)
    c.q, c.k, c.v, c.pos, c.slots = c.q[:0], c.k[:0], c.v[:0], c.pos[:0], c.slots[:0]
    was = c.kp.clone()
    assert c.run().shape == (0, 8, 64) and torch.equal(c.kp, was)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_one_weight_only_and_fp32_weights(dev, dtype):
    c = Case(dev, N=21, dtype=dtype, norm32=True, eps=0.0)
    c.check()
    c.qn = None
    c.check()
    c.qn, c.kn = c.kn.to(dtype), None
    c.check()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sizes_of_the_values(dev, dtype):
    """Tiny and huge rows, and rows of zeros, which stay zeros."""
    c = Case(dev, N=6, dtype=dtype, eps=1e-6)
    for t in (c.q, c.k):
        t[0] *= 2.0 ** -12
        t[1] = 0
        t[2] *= 2.0 ** 9
    c.check()


@pytest.mark.parametrize("long", [True, False])
def test_rows_that_are_not_kept_and_positions_outside(dev, long):
    c = Case(dev, N=9, long=long, norm=False, R=32)
    P = c.kp.shape[0]
    c.slots[2], c.slots[5], c.slots[7] = -1, P * 16, 2 ** 40
    c.check()
    bad = (0, 4, 8)
    c.pos[0], c.pos[4], c.pos[8] = -1, 500, 2 ** 31 - 1
    if long:
        c.pos[8] = 2 ** 50
    out = c.run()
    for i in range(9):
        s = int(c.slots[i])
        rows = [out[i]] + ([c.kp[s // 16, :, s % 16]] if 0 <= s < P * 16 else [])
        for row in rows:
            assert bool(torch.isnan(row[..., :32]).all()) == (i in bad) and not bool(torch.isnan(row[..., 32:]).any())
    assert torch.equal(out[bad, :, 32:], c.q[bad, :, 32:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lead", [1, 8])
def test_strides(dev, dtype, lead):
    """Rows at any element; a call copies those that are not 16-byte aligned."""
    Case(dev, N=30, dtype=dtype, lead=lead).check()
    c = Case(dev, N=30, dtype=dtype)
    c.q = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    c.k = c.k.repeat(1, 1, 2)[..., ::2].contiguous().flip(1)
    c.v = torch.cat([c.v, c.v], 2)[..., ::2]
    c.kp = c.kp.transpose(1, 2).contiguous().transpose(1, 2)
    c.vp = c.vp.transpose(1, 2).contiguous().transpose(1, 2)
    c.check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("form", ["new", "given", "odd", "itself"])
def test_outputs(dev, dtype, form):
    c = Case(dev, N=40, H=6, Hk=2, dtype=dtype, seed=2)
    want = c.run()
    if form == "given":
        out = torch.zeros(40, 12, 64, dtype=dtype, device=dev)[:, ::2]
    elif form == "odd":
        out = torch.zeros(40, 6, 65, dtype=dtype, device=dev)[..., 1:]
    else:
        out = c.q if form == "itself" else None
    got = c.run(out=out)
    assert torch.equal(got, want) and (out is None or got is out)


def test_replays_and_streams(dev):
    c = Case(dev, N=70, D=128)
    want = c.run()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    kp = c.kp.clone()
    c.kp.zero_()
    torch.cuda.synchronize()
    got = c.run(stream=s)
    torch.cuda.synchronize()
    rows = lambda t: t[c.slots // 16, :, c.slots % 16]  # noqa: E731
    assert torch.equal(got, want) and torch.equal(rows(c.kp), rows(kp))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.run()
    for i in range(3):
        c.pos.copy_((c.pos + 17) % 500)
        c.slots.copy_(c.slots.flip(0))
        out.zero_()
        graph.replay()
        c.check(out)
        assert torch.equal(out, c.run())


def test_slots_past_32_bit_offsets(dev):
    c = Case(dev, N=3, H=2, Hk=1, D=128, bs=64, dtype=BF16)
    P = (2 ** 32 + 2 ** 20) // (64 * 128)
    c.kp = torch.zeros((P, 1, 64, 128), dtype=BF16, device=dev)
    c.vp = torch.zeros_like(c.kp)
    c.slots = torch.tensor([P * 64 - 1, 5, P * 64 - 70], device=dev)
    c.run()
    for t, new in ((c.vp, c.v),):
        for i, s in enumerate(c.slots.tolist()):
            assert torch.equal(t[s // 64, :, s % 64], new[i])
    assert math.isclose(float((c.vp != 0).sum()), float((c.v != 0).sum()))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("norm32", [False, True])
def test_weights_that_begin_anywhere(dev, dtype, norm32):
    c = Case(dev, N=23, D=128, dtype=dtype, norm32=norm32, pairs=True, R=48)
    wide = torch.zeros(300, dtype=c.qn.dtype, device=dev)
    wide[1:129], wide[133:261] = c.qn, c.kn
    c.qn, c.kn = wide[1:129], wide[133:261]
    c.check()


def test_tables_of_cosines_that_begin_anywhere(dev):
    c = Case(dev, N=9, R=32)
    wide = [torch.zeros(c.cos.numel() + 3, device=dev) for _ in range(2)]
    for w, t in zip(wide, (c.cos, c.sin)):
        w[3:] = t.reshape(-1)
    c.cos, c.sin = (w[3:].view(500, 16) for w in wide)
    c.check()


def test_a_stores_rows_stay_where_blocks_move(dev):
    """TieredStorage.rotate_rows: the blocks written are the GPU tier's again, at once and after a move back."""
    from halo_amd import TieredStorage
    c = Case(dev, N=5, H=4, Hk=2, D=64, bs=4)
    st = TieredStorage(tiers=["gpu", "dram"], num_layers=2, num_kv_heads=2, head_dim=64, block_size=4, dtype=BF16, device=dev,
                       max_blocks=8)
    for layer in range(2):
        for b in range(8):
            st.write_new_block(layer=layer, block=b, keys=torch.full((2, 4, 64), float(b), device=dev),
                               values=torch.full((2, 4, 64), 100.0 + b, device=dev))
        st.move_blocks(layer=layer, blocks=torch.arange(1, 8, dtype=torch.int32, device=dev), src="gpu", dst="dram")
    slots = torch.tensor([9, -1, 10, 20, 2 ** 34], device=dev)
    want = c.run()  # the same rows in another pool
    rows = [c.kp[s // 4, :, s % 4].clone() for s in c.slots.tolist()]
    q = st.rotate_rows(q=c.q, keys=c.k, values=c.v, positions=c.pos, cos=c.cos, sin=c.sin, slots=slots, layer=1, q_norm=c.qn,
                       k_norm=c.kn)
    assert torch.equal(q, want)
    assert st.directory().tolist() == [[0] + [1] * 7, [0, 1, 0, 1, 1, 0, 1, 1]]
    for again in (False, True):
        for b, r, n in ((2, 1, 0), (2, 2, 2), (5, 0, 3)):
            kb, vb = st.read_block(layer=1, block=b)
            assert torch.equal(kb[:, r], rows[n]) and torch.equal(vb[:, r], c.v[n])
        kb, _ = st.read_block(layer=1, block=2)
        assert bool((kb[:, [0, 3]] == 2).all())
        st.move_blocks(layer=1, blocks=torch.arange(8, dtype=torch.int32, device=dev), src="dram", dst="gpu")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("D,R", [(64, 32), (128, 16), (128, 112)])
def test_channels_that_do_not_rotate_meet_no_others(dev, D, R, pairs, dtype):
    """An infinity or NaN behind the first R channels stays where it is; the others, zeros of either sign too, are the input's."""
    c = Case(dev, N=70 if D == 64 else 1400, D=D, R=R, dtype=dtype, pairs=pairs, norm=False, seed=R)  # few heads and many
    want, rows = c.run(), lambda t: t[c.slots // 16, :, c.slots % 16]
    k_want = rows(c.kp)
    for t in (c.q, c.k):
        t[..., R + 1], t[..., R + 4] = -0.0, 0.0
        t[0:60:3, :, R + 3] = float("inf")
        t[1:60:3, :, D - 1] = float("nan")
        t[2:60:3, :, R + 9] = -float("inf")
    out = c.run()
    for got, x, ref in ((out, c.q, want), (rows(c.kp), c.k, k_want)):
        tail = x[..., R:]
        assert torch.equal(got[..., R:].nan_to_num(nan=7.0), tail.nan_to_num(nan=7.0))
        assert torch.equal(torch.isnan(got[..., R:]), torch.isnan(tail))
        there = ~torch.isnan(tail)
        assert torch.equal(torch.signbit(got[..., R:])[there], torch.signbit(tail)[there])
        assert torch.equal(got[..., :R], ref[..., :R])
