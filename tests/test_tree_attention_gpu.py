"""Attention of drafted trees over a paged cache on the GPU, against the
definition in float64.

Tolerances, per element, with u the unit roundoff of fp32 (2^-24), A the
weighted mean of |v|, d the largest scale * sum |q_d k_d| of an attended row, T
the attended rows:
  scores  D products and sums, the scale and the exponent's fma:  (D + 6) u d
  exp2    one ulp:                                                2 u
  sums    of weights and of weighted values, in any order:        T u each
  weights rounded to a 16-bit pool's type:                        half a step
          (bf16 2^-8, fp16 2^-11) of each; below fp16's normal range at most
          2^-25 of the largest weight, which is at least 1
  out     rounded to its type:                                    half a step of |out|
so |out - exact| <= A (2 (D + 6) u d + (2 T + 8) u + w) + T 2^-25 max|v| [fp16] + r |out|
and |lse - exact| <= (D + 6) u d + (T + 8) u + 4 u |lse|.
"""
from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Case:
    """A batch: pools with blocks in random order, everything behind the requests' rows NaN."""

    def __init__(self, dev, *, lengths, nodes, H=8, Hk=2, D=64, bs=16, dtype=torch.bfloat16, tree="tree", seed=0,
                 sigma=1.0, spare=3, wide=2):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.dev, self.dtype, self.D, self.bs, self.H = dev, dtype, D, bs, H
        self.lengths, self.nodes = list(lengths), list(nodes)
        B = len(lengths)
        need = [-(-(c + n) // bs) for c, n in zip(lengths, nodes)]
        W = max(max(need), 1) + wide
        ids = list(range(sum(need) + spare))
        rng.shuffle(ids)
        P = len(ids)
        self.table = [[-1] * W for _ in range(B)]
        self.k = torch.full((P, Hk, bs, D), math.nan)
        self.v = torch.full((P, Hk, bs, D), math.nan)
        for b in range(B):
            self.table[b][:need[b]] = [ids.pop() for _ in range(need[b])]
            for p in range(lengths[b] + nodes[b]):
                x, r = self.table[b][p // bs], p % bs
                self.k[x, :, r] = torch.randn(Hk, D, generator=g)
                self.v[x, :, r] = torch.randn(Hk, D, generator=g)
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
        N = self.cu[-1]
        self.q = torch.randn(N, H, D, generator=g) * sigma
        self.max_nodes = max(max(nodes), 1)
        self.trees = []
        for n in nodes:
            self.trees.append([rng.randint(max(-1, i - 7), i - 1) for i in range(n)] if tree == "tree"
                              else list(range(-1, n - 1)))
        self.sees = [s for t in self.trees for s in paged.ancestors(t)]
        self.masks = tree != "causal"
        self.scale = D ** -0.5

    def device(self):
        d = self.dev
        words = -(-self.max_nodes // 64)
        return dict(q=self.q.to(self.dtype).to(d), k_pool=self.k.to(self.dtype).to(d), v_pool=self.v.to(self.dtype).to(d),
                    block_table=_i32(self.table, d), lengths=_i32(self.lengths, d), cu_nodes=_i32(self.cu, d),
                    mask=torch.from_numpy(paged.words(self.sees, words)).to(d) if self.masks else None,
                    max_nodes=self.max_nodes)

    def exact(self):
        f = [x.to(self.dtype).double().numpy() for x in (self.q, self.k, self.v)]
        return paged.attend(*f, self.table, self.lengths, self.cu, self.sees, self.scale)

    def rows(self):
        return max([c + n for c, n in zip(self.lengths, self.nodes)])

    def check(self, out, lse, exact=None, out_dtype=None):
        ref, rl, mean, dots = self.exact() if exact is None else exact
        T, D = self.rows(), self.D
        w = 0.0 if self.dtype == torch.float32 else HALF[self.dtype]
        tol = mean * (2 * (D + 6) * U * dots[..., None] + (2 * T + 8) * U + w)
        if self.dtype == torch.float16:
            tol = tol + T * 2.0 ** -25 * float(np.nanmax(np.abs(self.v.numpy())))
        tol = tol + HALF[out_dtype or self.dtype] * np.abs(ref) * (1 + w)
        o = out.double().cpu().numpy()
        fine = np.isfinite(ref)
        assert np.array_equal(np.isnan(o), np.isnan(ref)) and np.array_equal(o[~fine & ~np.isnan(ref)],
                                                                             ref[~fine & ~np.isnan(ref)])
        with np.errstate(invalid="ignore"):
            worst = np.where(fine, np.abs(o - ref) - tol, -1)
        assert worst.max() <= 0, f"off by {worst.max():.3e} more than allowed at {np.unravel_index(worst.argmax(), o.shape)}"
        z = lse.double().cpu().numpy()
        none = np.isneginf(rl)
        assert np.array_equal(np.isneginf(z), none)
        with np.errstate(invalid="ignore"):
            lt = (D + 6) * U * dots + (T + 8) * U + 4 * U * np.abs(rl)
            assert (np.abs(z - rl)[~none & np.isfinite(rl)] <= lt[~none & np.isfinite(rl)]).all()


def _run(c, **kw):
    import halo_amd
    return halo_amd.tree_attention(**{**c.device(), **kw}, return_lse=True)


DT = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths,nodes", [([0], [1]), ([1], [1]), ([31], [1]), ([32], [2]), ([33], [7]), ([100], [33]),
                                           ([257], [64]), ([700], [65]), ([5, 0, 300], [3, 1, 20])])
def test_small_batches(dev, dtype, D, lengths, nodes):
    c = Case(dev, lengths=lengths, nodes=nodes, D=D, dtype=dtype, seed=len(nodes) + lengths[0])
    c.check(*_run(c))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("bs", [1, 3, 8, 16, 24, 32, 64, 100, 256])
def test_block_sizes(dev, dtype, bs):
    c = Case(dev, lengths=[211, 3, 64], nodes=[9, 4, 12], bs=bs, dtype=dtype, seed=bs)
    c.check(*_run(c))


@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 8), (28, 4), (32, 8), (6, 2), (40, 1), (64, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_head_layouts(dev, dtype, H, Hk):
    c = Case(dev, lengths=[150, 37], nodes=[11, 5], H=H, Hk=Hk, D=128, dtype=dtype, seed=H)
    c.check(*_run(c))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lengths,nodes", [([2500], [17]), ([4100, 1, 900], [8, 20, 1])])
def test_long_requests_are_cut_and_merged(dev, dtype, lengths, nodes):
    c = Case(dev, lengths=lengths, nodes=nodes, H=4, Hk=2, D=128, dtype=dtype, seed=5)
    c.check(*_run(c))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_large_trees(dev, dtype):
    c = Case(dev, lengths=[40, 0], nodes=[512, 130], H=2, Hk=1, D=64, dtype=dtype, seed=6)
    c.check(*_run(c))


@pytest.mark.parametrize("nodes", [[1], [70, 3], [200]])
def test_without_masks_the_rows_are_causal(dev, nodes):
    c = Case(dev, lengths=[90, 12][:len(nodes)], nodes=nodes, tree="causal", dtype=torch.bfloat16, seed=7)
    c.check(*_run(c))


def test_many_requests(dev):
    rng = random.Random(8)
    n = [rng.choice([0, 0, 1, 2, 5]) for _ in range(150)]
    c = Case(dev, lengths=[rng.choice([0, 1, 20, 60]) for _ in n], nodes=n, H=2, Hk=1, D=64, dtype=torch.float16, seed=8)
    c.check(*_run(c))


@pytest.mark.parametrize("dtype,nodes", [(torch.float16, 2), (torch.bfloat16, 40), (torch.float32, 3)])
def test_hundreds_of_requests_some_of_them_long(dev, dtype, nodes):
    rng = random.Random(23)
    B = 300
    ln = [rng.choice([0, 3, 40]) for _ in range(B)]
    n = [rng.choice([0, 1, nodes]) for _ in range(B)]
    for b in (0, 63, 64, 255, 256, 299):  # cut requests on both sides of what one look covers
        ln[b], n[b] = 1200 + b, nodes
    c = Case(dev, lengths=ln, nodes=n, H=2, Hk=1, D=64, dtype=dtype, seed=23)
    c.check(*_run(c))


@pytest.mark.parametrize("dtype,nodes", [(torch.bfloat16, 3), (torch.float16, 30), (torch.float32, 2)])
def test_a_long_request(dev, dtype, nodes):
    c = Case(dev, lengths=[40003], nodes=[nodes], H=4, Hk=1, D=64, dtype=dtype, seed=24)
    c.check(*_run(c))


@pytest.mark.parametrize("dtype", DT)
def test_large_scores(dev, dtype):
    """Scores of several hundred: the running maximum moves and small weights vanish."""
    c = Case(dev, lengths=[400], nodes=[6], D=128, dtype=dtype, sigma=30.0, seed=9)
    c.check(*_run(c))


@pytest.mark.parametrize("dtype", DT)
def test_rows_that_see_nothing(dev, dtype):
    c = Case(dev, lengths=[0, 50, 0], nodes=[5, 2, 40], dtype=dtype, seed=10)
    c.sees[1] = set()
    c.sees[2] = {0, 4}
    for i in range(7, 47):
        c.sees[i] = set() if i % 3 else {i - 7}
    out, lse = _run(c)
    c.check(out, lse)
    assert not out[1].any() and bool((lse[1] == -math.inf).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_not_finite_reach_only_the_nodes_that_see_them(dev, dtype, D):
    c = Case(dev, lengths=[37], nodes=[40], H=4, Hk=2, D=D, dtype=dtype, seed=11, tree="tree")
    for p, val in ((37 + 3, math.nan), (37 + 8, math.inf), (37 + 9, -math.inf), (37 + 33, math.inf)):
        x, r = c.table[0][p // c.bs], p % c.bs
        c.v[x, :, r, ::3] = val
    for p, val in ((37 + 5, math.nan), (37 + 12, math.inf)):
        x, r = c.table[0][p // c.bs], p % c.bs
        c.k[x, 1, r, 7] = val
    c.sees = [s - {12} if i != 12 else s for i, s in enumerate(c.sees)]
    out, lse = _run(c)
    ref, rl, *_ = ex = c.exact()
    touched = [i for i, s in enumerate(c.sees) if s & {5, 12}]
    keep = [i for i in range(40) if i not in touched]
    assert len(keep) > 20 and np.isnan(ref[keep]).any() and np.isinf(ref[keep]).any()
    got = out.double().cpu().numpy()
    assert np.array_equal(np.isnan(got[keep]), np.isnan(ref[keep]))
    sub = tuple(x[keep] for x in ex)
    c.check(out[keep], lse[keep], exact=sub)
    sees5 = [i for i, s in enumerate(c.sees) if 5 in s]
    assert np.isnan(got[sees5, 2:]).all() and torch.isnan(lse[sees5, 2:]).all()  # the heads of KV head 1


@pytest.mark.parametrize("dtype", DT)
def test_rows_in_blocks_outside_the_pool_are_not_attended(dev, dtype):
    c = Case(dev, lengths=[300, 60], nodes=[9, 4], dtype=dtype, seed=12)
    P = c.k.shape[0]
    c.table[0][3], c.table[0][7], c.table[0][8], c.table[1][0] = -1, P, 2 ** 31 - 1, -2 ** 31
    c.check(*_run(c))


def test_table_that_ends_before_the_rows(dev):
    c = Case(dev, lengths=[100], nodes=[6], seed=13, wide=0)
    c.table = [c.table[0][:6]]  # 96 of the 106 rows
    c.check(*_run(c))


def test_nodes_past_max_nodes_and_padding_are_left_out(dev):
    c = Case(dev, lengths=[20, 30], nodes=[6, 3], seed=14)
    d = c.device()
    q = torch.cat([d["q"], torch.full((4,) + d["q"].shape[1:], math.nan, device=dev, dtype=c.dtype)])
    mask = torch.cat([d["mask"], d["mask"].new_zeros(4, 1)])
    out = torch.full(q.shape, 7.0, device=dev, dtype=c.dtype)
    lse = torch.full(q.shape[:2], 8.0, device=dev)
    _run(c, q=q, mask=mask, out=out, lse=lse, max_nodes=4)
    c.sees = [s & set(range(4)) for s in c.sees]
    ref = tuple(np.concatenate([x[:4], x[6:]]) for x in c.exact())
    c.check(torch.cat([out[:4], out[6:9]]), torch.cat([lse[:4], lse[6:9]]), exact=ref)
    assert bool((out[4:6] == 7).all()) and bool((out[9:] == 7).all())
    assert bool((lse[4:6] == 8).all()) and bool((lse[9:] == 8).all())


def test_longer_masks_than_needed(dev):
    c = Case(dev, lengths=[20], nodes=[6], seed=15)
    m = torch.cat([c.device()["mask"], torch.full((6, 2), -1, dtype=torch.int64, device=dev)], 1)
    c.check(*_run(c, mask=m))


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float16),
                                             (torch.float16, torch.bfloat16)])
def test_out_dtype(dev, dtype, out_dtype):
    c = Case(dev, lengths=[70], nodes=[4], dtype=dtype, seed=16)
    out, lse = _run(c, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    c.check(out, lse, out_dtype=out_dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(dev, dtype):
    """q as a slice of a projection and at an odd start, pools with the rows outside the heads, out in wider rows."""
    c = Case(dev, lengths=[70, 9], nodes=[4, 3], dtype=dtype, seed=17)
    ex, d = c.exact(), c.device()
    kp, vp = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (d["k_pool"], d["v_pool"]))
    wide = torch.empty(7, 3, c.H, c.D, device=dev, dtype=dtype)
    wide[:, 1] = d["q"]
    odd = torch.empty(7, c.H, c.D + 1, device=dev, dtype=dtype)
    odd[..., 1:] = d["q"]
    for q in (wide[:, 1], odd[..., 1:], d["q"].transpose(0, 1).contiguous().transpose(0, 1)):
        for o in (torch.empty(7, c.H + 2, c.D + 3, device=dev, dtype=dtype)[:, 1:-1, 1:-2],
                  torch.empty(7, c.H + 2, c.D, device=dev, dtype=dtype)[:, 2:]):
            out, lse = _run(c, q=q, k_pool=kp, v_pool=vp, out=o)
            assert out is o
            c.check(out, lse, exact=ex)


def test_scale(dev):
    c = Case(dev, lengths=[70], nodes=[4], seed=18)
    for s in (1.0, 1e-30, 0.02):
        c.scale = s
        c.check(*_run(c, scale=s))


def test_two_calls_agree_bit_for_bit_and_with_another_batch_around(dev):
    c = Case(dev, lengths=[900, 20], nodes=[5, 9], D=128, seed=19)
    a, b = _run(c), _run(c)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_on_another_stream(dev):
    c = Case(dev, lengths=[500, 33], nodes=[5, 9], D=128, seed=20)
    ex = c.exact()
    d = c.device()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    out, lse = _run(c, stream=s, **d)
    s.synchronize()
    c.check(out, lse, exact=ex)


def test_captured_call_follows_lengths_and_trees(dev):
    """One graph, replayed between eager work with other lengths, trees and tables in the same tensors."""
    import halo_amd
    cases = [Case(dev, lengths=ln, nodes=n, H=4, Hk=2, D=64, seed=21 + i, spare=200 - sum(-(-(a + b) // 16) for a, b in zip(ln, n)))
             for i, (ln, n) in enumerate([([900, 20], [5, 9]), ([0, 1500], [1, 13]), ([300, 300], [12, 0])])]
    size = [max(c.device()[k].shape[0] for c in cases) for k in ("q",)][0]
    W = max(len(c.table[0]) for c in cases)
    dev_ = dict(q=torch.zeros(size, 4, 64, device=dev, dtype=torch.bfloat16),
                k_pool=torch.zeros_like(cases[0].device()["k_pool"]), v_pool=torch.zeros_like(cases[0].device()["v_pool"]),
                block_table=torch.full((2, W), -1, dtype=torch.int32, device=dev), lengths=_i32([0, 0], dev),
                cu_nodes=_i32([0, 0, 0], dev), mask=torch.zeros(size, 1, dtype=torch.int64, device=dev))
    out = torch.zeros(size, 4, 64, device=dev, dtype=torch.bfloat16)
    lse = torch.zeros(size, 4, device=dev)

    def fill(c):
        for k, t in c.device().items():
            if k == "block_table":
                dev_[k].fill_(-1)
                dev_[k][:, :t.shape[1]] = t
            elif torch.is_tensor(t):
                dev_[k][:t.shape[0]] = t

    fill(cases[0])
    call = lambda: halo_amd.tree_attention(**dev_, max_nodes=13, out=out, lse=lse)  # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call()
    for c in cases + cases[::-1]:
        fill(c)
        g.replay()
        n = c.cu[-1]
        got = out[:n].clone(), lse[:n].clone()
        call()
        assert torch.equal(got[0], out[:n]) and torch.equal(got[1], lse[:n])
        c.check(*got)


def test_two_graphs_replayed_in_turn(dev):
    """Each captured call has partials of its own."""
    import halo_amd
    cs = [Case(dev, lengths=[2000], nodes=[5], H=4, Hk=2, D=128, seed=25),
          Case(dev, lengths=[1500, 700], nodes=[30, 11], H=4, Hk=2, D=128, seed=26)]
    args = [c.device() for c in cs]
    want = [halo_amd.tree_attention(**a, return_lse=True) for a in args]
    graphs, got = [], []
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            got.append(halo_amd.tree_attention(**a, return_lse=True))
        graphs.append(g)
    for i in (0, 1, 1, 0, 1, 0):
        graphs[i].replay()
        junk = torch.full((1 << 20,), math.nan, device=dev)  # eager work between the replays
        for a, b in zip(got[i], want[i]):
            assert torch.equal(a, b)
        del junk


def test_offsets_past_32_bits(dev):
    """The same blocks at the far end of pools of 5.6 GB give the same bits."""
    import halo_amd
    c = Case(dev, lengths=[100, 300], nodes=[9, 40], H=32, Hk=8, D=128, seed=27, spare=0)
    a = c.device()
    k = torch.randn(5, 8, 128, device=dev).to(c.dtype)
    P, far = a["k_pool"].shape[0], 170000
    big = [torch.empty(far + P, 8, 16, 128, device=dev, dtype=c.dtype) for _ in range(2)]
    assert big[0].numel() > 2 ** 31
    slots = torch.tensor([3, 17, 40, 41, 60], device=dev)
    path, n_path = _i32([[0, 2, 5], [1, 4, 9]], dev), _i32([3, 3], dev)
    outs = []
    for kp, vp, off in ((a["k_pool"], a["v_pool"], 0), (big[0], big[1], far)):
        if off:
            kp[far:], vp[far:] = keep
        else:
            keep = kp.clone(), vp.clone()
        t = torch.where(a["block_table"] >= 0, a["block_table"] + off, -1).int()
        halo_amd.append_rows(k, -k, slots + off * 16, kp, vp)
        d = {**a, "k_pool": kp, "v_pool": vp, "block_table": t}
        out, lse = halo_amd.tree_attention(**d, return_lse=True)
        new = halo_amd.commit_path(kp, vp, t, a["lengths"], path, n_path)
        outs.append([out, lse, new, kp[off:].clone().view(torch.int16), vp[off:].clone().view(torch.int16)])
    for x, y in zip(*outs):
        assert torch.equal(x.nan_to_num(7) if x.is_floating_point() else x, y.nan_to_num(7) if y.is_floating_point() else y)


def test_speculative_steps_together(dev):
    """Three steps of a batch: room, layout, rows, attention of two layers, a path kept; against the same done row by row."""
    import halo_amd
    from halo_amd import TieredStorage
    rng = random.Random(22)
    B, H, Hk, D, bs, Lr, dt = 3, 4, 2, 64, 8, 2, torch.float16
    st = TieredStorage(tiers=["gpu"], num_layers=Lr, num_kv_heads=Hk, head_dim=D, block_size=bs, dtype=dt, device=dev,
                       max_blocks=60)
    kp, vp = st.pool()
    kp.fill_(math.nan)
    vp.fill_(math.nan)
    table = torch.full((B, 16), -1, dtype=torch.int32, device=dev)
    owned, free, n_free = _i32([0] * B, dev), _i32(rng.sample(range(60), 60), dev), _i32([60], dev)
    lengths = _i32([0] * B, dev)
    kept = [[([], []) for _ in range(Lr)] for _ in range(B)]  # committed rows, row by row
    for step in range(4):
        ctx = [len(kept[b][0][0]) for b in range(B)]
        assert lengths.tolist() == ctx
        sizes = [rng.randint(1, 30) for _ in range(B)]
        trees = [list(range(-1, n - 1)) if step == 0 else [rng.randint(max(-1, i - 4), i - 1) for i in range(n)] for n in sizes]
        N = sum(sizes)
        new = _i32([c + n for c, n in zip(ctx, sizes)], dev)
        up = halo_amd.update_block_tables(table, owned, free, n_free, new, lengths, block_size=bs, max_rows=N)
        assert bool(up.ok.all())
        mask, depth = halo_amd.tree_layout(_i32(sum(trees, []), dev), up.cu_rows, max_nodes=max(sizes))
        cu = up.cu_rows.tolist()
        sets = [s for t in trees for s in paged.ancestors(t)]
        k, v = (torch.randn(Lr, N, Hk, D, device=dev).to(dt) for _ in range(2))
        for layer in range(Lr):
            halo_amd.append_rows(k[layer], v[layer], up.slots, kp[layer], vp[layer])
            q = torch.randn(N, H, D, device=dev).to(dt)
            out, lse = halo_amd.tree_attention(q, kp[layer], vp[layer], table, lengths, up.cu_rows, mask=mask,
                                               max_nodes=max(sizes), return_lse=True)
            for b in range(B):
                rk = kept[b][layer][0] + list(k[layer, cu[b]:cu[b + 1]])
                rv = kept[b][layer][1] + list(v[layer, cu[b]:cu[b + 1]])
                flat = (torch.stack(rk).transpose(0, 1)[None].double().cpu().numpy(),
                        torch.stack(rv).transpose(0, 1)[None].double().cpu().numpy())
                c = Case(dev, lengths=[ctx[b]], nodes=[sizes[b]], H=H, Hk=Hk, D=D, dtype=dt)
                c.v = torch.stack(rv).float().cpu()
                ex = paged.attend(q[cu[b]:cu[b + 1]].double().cpu().numpy(), *[x.reshape(1, Hk, -1, D) for x in flat], [[0]],
                                  [ctx[b]], [0, sizes[b]], sets[cu[b]:cu[b + 1]], D ** -0.5)
                c.check(out[cu[b]:cu[b + 1]], lse[cu[b]:cu[b + 1]], exact=ex)
        paths = []
        for n, t in zip(sizes, trees):
            leaf = rng.randrange(n)
            paths.append(sorted(paged.ancestors(t)[leaf]) if step else list(range(min(n, 64))))
        P = max(len(p) for p in paths)
        lengths = halo_amd.commit_path(kp, vp, table, lengths, _i32([p + [0] * (P - len(p)) for p in paths], dev),
                                       _i32([len(p) for p in paths], dev))
        for b in range(B):
            for layer in range(Lr):
                kept[b][layer][0].extend(k[layer, cu[b] + i] for i in paths[b])
                kept[b][layer][1].extend(v[layer, cu[b] + i] for i in paths[b])
    zero = _i32([0] * B, dev)
    halo_amd.update_block_tables(table, owned, free, n_free, zero, zero, block_size=bs, max_rows=0)
    assert sorted(free.tolist()) == list(range(60)) and n_free.tolist() == [60] and not owned.any()
