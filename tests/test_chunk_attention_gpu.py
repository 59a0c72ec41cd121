"""Chunks attended over a paged cache on the GPU, against the definition in
float64 (tree_launch.Batch without masks).

Tolerances as in test_tree_pipeline_gpu.py, with u = 2^-24, A the weighted mean
of |v|, d the largest scale * sum |q_d k_d|, T the attended rows:
  |out - exact| <= A (2 (D + 6) u d + (2 T + 8) u + w) + f + r |out| (1 + w)
  |lse - exact| <= (D + 6) u d + (T + 8) u + 4 u |lse|"""
from __future__ import annotations

import copy

import pytest
import torch

import tree_launch
from test_tree_pipeline_gpu import BF16, F16, F32, HALF, U, check

pytestmark = pytest.mark.gpu
DT = [BF16, F16, F32]


class Batch(tree_launch.Batch):
    def __init__(self, dev, **kw):
        super().__init__(dev, **{**dict(H=8, Hk=2, D=64, bs=16, dtype=BF16, seed=0, blocks=200), **kw}, masks=False)

    def exact(self, only=None):
        return super().exact([b for b, n in enumerate(self.nodes) if n] if only is None else only)

    def run(self, **kw):
        import halo_amd
        a = dict(self.args)
        a.pop("mask")
        a["cu_rows"] = a.pop("cu_nodes")
        return halo_amd.chunk_attention(**{**a, **dict(max_rows=self.max_nodes, return_lse=True), **kw})


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx,rows", [(0, 1), (5, 1), (0, 64), (100, 256), (3, 257), (0, 512), (1, 514), (63, 577), (64, 1023),
                                      (700, 640), (31, 1025), (5000, 300)])
def test_one_request(dev, ctx, rows, D, dtype):
    b = Batch(dev, lengths=[ctx], nodes=[rows], D=D, dtype=dtype, seed=rows)
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 8), (28, 4), (32, 8), (6, 2), (40, 1), (24, 1)])
def test_head_layouts(dev, dtype, H, Hk):
    b = Batch(dev, lengths=[37, 0, 300], nodes=[600, 1, 77], H=H, Hk=Hk, D=128, dtype=dtype, seed=H)
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("holes", [0.0, 0.06])
@pytest.mark.parametrize("bs", [1, 3, 16, 24, 100, 256])
def test_blocks_of_any_size_and_blocks_that_are_not_there(dev, bs, holes, dtype):
    b = Batch(dev, lengths=[1500, 0, 64], nodes=[530, 700, 2], bs=bs, holes=holes, dtype=dtype, seed=bs)
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("dtype", DT)
def test_ragged_batches(dev, dtype):
    """Empty requests, single rows behind long contexts, and prompts from nothing."""
    lengths = [0, 4000, 17, 0, 900, 2500, 0, 1, 64, 0]
    rows = [1200, 1, 0, 513, 64, 2, 0, 33, 640, 1]
    for H, Hk, D in ((8, 2, 64), (28, 4, 128)):
        b = Batch(dev, lengths=lengths, nodes=rows, H=H, Hk=Hk, D=D, dtype=dtype, seed=H)
        check(b, *b.run(), b.exact())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_contexts_cut_into_many_parts(dev, dtype):
    b = Batch(dev, lengths=[30000], nodes=[520], H=4, Hk=1, D=128, dtype=dtype, seed=3)
    check(b, *b.run(), b.exact())
    b = Batch(dev, lengths=[20000, 100], nodes=[513, 900], H=8, Hk=2, D=64, dtype=dtype, seed=4)
    check(b, *b.run(), b.exact())


def test_a_long_prompt(dev):
    b = Batch(dev, lengths=[0], nodes=[5000], H=4, Hk=1, D=128, dtype=BF16, seed=5)
    check(b, *b.run(), b.exact())
    b = Batch(dev, lengths=[11], nodes=[3001], H=2, Hk=2, D=64, dtype=F32, seed=5)
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("B", [65, 700, 4096])
def test_many_requests(dev, B):
    rows = [513 if b == 40 else (b * 7) % 4 for b in range(B)]
    b = Batch(dev, lengths=[(b * 13) % 90 for b in range(B)], nodes=rows, H=4, Hk=2, dtype=BF16, seed=B)
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("dtype", DT)
def test_few_rows_are_the_causal_tree(dev, dtype):
    """Up to 256 rows in all, by the same kernels; more rows, and so other kernels, give the same up to rounding."""
    b = Batch(dev, lengths=[300, 0, 1000], nodes=[40, 215, 1], dtype=dtype)
    got, want = b.run(), tree_launch.Batch.run(b)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for most in (100000, 2 ** 31 + 5, 2 ** 40):
        got = b.run(max_rows=most)
        check(b, *got, b.exact())
        assert torch.equal(got[0], b.run(max_rows=most, stream=torch.cuda.current_stream())[0])
    b = Batch(dev, lengths=[300, 0, 1000], nodes=[40, 216, 1], dtype=dtype)
    check(b, *b.run(), b.exact())
    check(b, *tree_launch.Batch.run(b), b.exact())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_are_not_seen_have_no_part(dev, dtype, value):
    """K and V behind a row, behind the request, and of blocks that no request has hold NaN or infinities."""
    ctx, n, bs, Hk, D = 70, 600, 16, 2, 64
    b = Batch(dev, lengths=[ctx], nodes=[n], dtype=dtype, seed=8)
    a = b.args
    a["block_table"][0] = torch.arange(b.W, device=dev)
    exact = b.exact()
    want = b.run()
    at = ctx + 333
    bounds = Batch(dev, lengths=[ctx], nodes=[n], dtype=dtype, seed=8)  # the values as they were
    for p in (a["k_pool"], a["v_pool"]):
        p[b.W:] = value
        p[-(-(ctx + n) // bs):] = value
        p[(ctx + n - 1) // bs, :, (ctx + n - 1) % bs + 1:] = value
    got = b.run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a["v_pool"][at // bs, :, at % bs, 5] = value  # a value that the rows from 333 on see
    out, lse = b.run()
    assert torch.equal(lse, want[1])
    keep = torch.ones(D, dtype=torch.bool, device=dev)
    keep[5] = False
    check(bounds, torch.where(torch.isfinite(out), out, want[0]), lse, exact)
    assert torch.equal(torch.isfinite(out)[..., 5], (torch.arange(n, device=dev) < 333)[:, None].expand(n, b.H))
    assert bool(torch.isfinite(out[..., keep]).all())
    a["k_pool"][at // bs, :, at % bs] = value  # and a key
    out, lse = b.run()
    assert bool(torch.isfinite(out[:333]).all()) and bool(torch.isfinite(lse[:333]).all())
    check(bounds, torch.where((torch.arange(n, device=dev) < 333)[:, None, None], out, want[0]),
          torch.where((torch.arange(n, device=dev) < 333)[:, None], lse, want[1]), exact)


def test_requests_without_any_row_there(dev):
    b = Batch(dev, lengths=[40, 10], nodes=[600, 20])
    b.args["block_table"][0] = -1
    out, lse = b.run()
    assert not bool(out[:600].any()) and bool((lse[:600] == -float("inf")).all())
    assert bool(torch.isfinite(lse[600:]).all())


def test_rows_behind_the_table(dev):
    """Lengths and rows past the table's columns are not attended and nothing is read there."""
    b = Batch(dev, lengths=[100], nodes=[600])
    a = b.args
    a["block_table"] = a["block_table"][:, :20].contiguous()
    out, lse = b.run()
    full = Batch(dev, lengths=[100], nodes=[600])
    want = full.run()
    assert torch.equal(out[:220], want[0][:220]) and torch.equal(lse[:220], want[1][:220])
    a["lengths"].fill_(2 ** 30)
    out, lse = b.run()
    assert bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("out_dtype", DT)
@pytest.mark.parametrize("form", ["plain", "odd start", "odd rows"])
def test_rows_of_no_request_keep_what_they_hold(dev, dtype, out_dtype, form):
    b = Batch(dev, lengths=[300, 20], nodes=[600, 3], dtype=dtype, seed=6)
    want = b.run()
    N = 607
    q = torch.cat([b.args["q"], b.args["q"][:4]])
    shape, cut = {"plain": ((N, 8, 64), slice(None)), "odd start": ((N, 8, 66), slice(1, 65)), "odd rows": ((N, 8, 65), slice(0, 64))}[form]
    held = (torch.arange(N * 8 * shape[2], device=dev, dtype=torch.float32).view(shape) % 251 - 125).to(out_dtype)
    out = held.clone()[..., cut]
    lse = torch.full((N, 8), 7.0, device=dev)
    got = b.run(q=q, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    assert torch.equal(out[603:], held[603:, :, cut]) and bool((lse[603:] == 7).all())
    full = b.run(out_dtype=F32)[0]
    # where a request is cut goes by the call's room for rows too, and so do its last bits
    tol = (HALF[out_dtype] + HALF[dtype]) * 2 * full.abs() + 1e-3 * (dtype != F32) + 1e-5
    assert bool(((out[:603].float() - full).abs() <= tol).all()) and torch.equal(full.to(dtype), want[0])
    # rows past max_rows are left out as well
    out = held.clone()[..., cut]
    b.run(q=q, out=out, lse=lse, max_rows=550)
    assert torch.equal(out[550:600], held[550:600, :, cut])


@pytest.mark.parametrize("dtype", DT)
def test_strides(dev, dtype):
    b = Batch(dev, lengths=[77, 0], nodes=[520, 9], dtype=dtype, seed=7)
    want = b.run()
    a = b.args
    q = a["q"]
    for form in (q.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([q, q], 2)[..., :64], torch.cat([q, q], 2)[..., 1:65].clone(),
                 torch.nn.functional.pad(q, (1, 0))[..., 1:]):
        if form.shape == q.shape and torch.equal(form, q):
            got = b.run(q=form)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    pools = [p.transpose(1, 2).contiguous().transpose(1, 2) for p in (a["k_pool"], a["v_pool"])]
    table = torch.nn.functional.pad(a["block_table"], (0, 5), value=-1)[:, :b.W]
    got = b.run(k_pool=pools[0], v_pool=pools[1], block_table=table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_scales(dev):
    b = Batch(dev, lengths=[10], nodes=[520], dtype=F32, seed=9)
    got = b.run(scale=0.5)
    b.args["q"] = b.args["q"] * (0.5 * 8.0)  # the default is 1 / 8
    want = b.run()
    assert float((got[0] - want[0]).abs().max()) < 1e-5


def test_replays_follow_the_lengths(dev):
    """One graph, batches of other lengths and rows; eager calls between the replays."""
    b = Batch(dev, lengths=[1000, 50, 3], nodes=[600, 40, 13], seed=10, blocks=100)
    a = b.args
    b.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = b.run()
    N = sum(b.nodes)
    for lengths, rows in (([1000, 50, 3], [600, 40, 13]), ([0, 500, 20], [1, 600, 52]), ([900, 0, 0], [0, 650, 3]),
                          ([1, 2, 3], [217, 217, 219])):
        b.lengths, b.nodes = lengths, rows
        rows = [min(r, 600) for r in rows]
        a["lengths"].copy_(torch.tensor(lengths))
        at = [0]
        for r in b.nodes:
            at.append(at[-1] + r)
        a["cu_nodes"].copy_(torch.tensor(at))
        out.fill_(5)
        graph.replay()
        eager = b.run()
        exact = b.exact()
        live = torch.cat([torch.arange(r, device=dev) < 600 for r in b.nodes])
        assert N == live.numel()
        assert torch.equal(out[live], eager[0][live]) and torch.equal(lse[live], eager[1][live])
        ref = [x[live] for x in exact]
        check(b, out[live], lse[live], ref)


def test_two_streams(dev):
    b1 = Batch(dev, lengths=[2000], nodes=[600], seed=1)
    b2 = Batch(dev, lengths=[30, 700], nodes=[700, 20], seed=2, dtype=F16)
    want = [b1.run(), b2.run()]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [b.run(stream=x) for b, x in zip((b1, b2), s)]
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_cu_rows_that_fall_or_pass_the_rows(dev):
    """Whatever cu_rows holds, no other memory is read or written: rows of more than one request get either's output."""
    b = Batch(dev, lengths=[10, 20, 30, 40], nodes=[600, 5, 600, 5])
    for cu in ([0, 1210, 0, 1210, 5000], [0, 600, 300, 1210, 1210], [-7, 2 ** 30, -2 ** 31, 2 ** 31 - 1, 0], [1210, 5, 4, 3, 2]):
        b.args["cu_nodes"].copy_(torch.tensor(cu))
        for most in (600, 300):
            out, lse = b.run(out=torch.zeros_like(b.args["q"]), max_rows=most)
            assert bool(torch.isfinite(out).all())


def test_huge_scores(dev):
    """The largest scores are about 5.2 standard deviations of 8 x 2^26 x scale.  fp16 is covered up to 2^24: from exponents of
    2^28 (steps of 32) the largest weight, rounded to a step of 2^7, may lie below 2^-14, where fp16 values lose bits."""
    for dtype in DT:
        b = Batch(dev, lengths=[700], nodes=[600], seed=3, dtype=dtype)
        for t in (b.args["q"], b.args["k_pool"]):
            t.mul_(2.0 ** 13).clamp_(-60000, 60000)
        b.args["v_pool"].abs_()
        out, lse = b.run(scale=2.0 ** (-8 if dtype == F16 else -3))
        top = float(b.args["v_pool"].max()) * (1 + 2 * HALF[dtype]) * (1 + 8000 * U)
        assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
        assert float(out.min()) >= 0 and float(out.max()) <= top


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("H,Hk,most", [(8, 2, 32), (8, 2, 33), (8, 2, 1), (28, 4, 18), (28, 4, 19), (8, 8, 128), (8, 8, 130), (40, 1, 3),
                                       (40, 1, 4)])
def test_batches_of_short_chunks(dev, dtype, H, Hk, most):
    """Around 128 rows of query heads a request, where 16-bit calls change kernels: also empty requests and single rows."""
    B = 1 + 2000 // (8 * most) * 8
    rows = [most if b % 3 == 0 else (b * 5) % (most + 1) for b in range(B)]
    rows[0] += max(0, 257 - sum(rows))  # more than 256 in all
    b = Batch(dev, lengths=[(b * 37) % 300 for b in range(B)], nodes=rows, H=H, Hk=Hk, dtype=dtype, seed=most)
    got = b.run(max_rows=max(rows))
    check(b, *got, b.exact())
    again = b.run(max_rows=max(rows), stream=torch.cuda.current_stream())
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    if dtype != F32 and max(rows) * (H // Hk) <= 128:
        want = tree_launch.Batch.run(b)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("H,Hk,B,most,trees", [(8, 2, 8, 48, True), (8, 2, 64, 64, True), (8, 2, 65, 64, False), (8, 2, 8, 65, False),
                                               (28, 4, 9, 36, True), (28, 4, 70, 36, False), (8, 8, 3, 256, True)])
def test_batches_of_up_to_a_unit(dev, dtype, H, Hk, B, most, trees):
    """Around 256 rows of query heads a request, and 16384 in all."""
    b = Batch(dev, lengths=[(k * 61) % 700 for k in range(B)], nodes=[most] * B, H=H, Hk=Hk, D=128, dtype=dtype, seed=B)
    assert trees == (most * H // Hk <= 256 and B * most * H // Hk <= 16384)
    got = b.run()
    check(b, *got, b.exact())
    if trees:
        want = tree_launch.Batch.run(b)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("most", [1, 3, 512])
def test_more_requests_than_a_plan_holds(dev, dtype, most):
    B = 4999
    rows = [most if b in (7, 4500) else (b * 7) % (min(most, 3) + 1) for b in range(B)]
    b = Batch(dev, lengths=[(b * 13) % 50 for b in range(B)], nodes=rows, H=4, Hk=2, dtype=dtype, seed=most)
    got = b.run()
    check(b, *got, b.exact())
    again = b.run(stream=torch.cuda.current_stream())
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_many_requests_of_many_rows_are_refused(dev):
    b = Batch(dev, lengths=[1] * 4097, nodes=[513] + [0] * 4096, H=4, Hk=2, seed=1)
    for kw in ({}, dict(stream=torch.cuda.current_stream())):
        with pytest.raises(Exception, match="4096"):
            b.run(**kw)
    b.run(max_rows=512)


def part_of(b, request, lo, n):
    """Rows lo .. lo + n - 1 of q as those of one request, alone."""
    c = copy.copy(b)
    c.lengths, c.nodes = [b.lengths[request]], [n]
    c.args = {**b.args, "q": b.args["q"][lo:lo + n], "block_table": b.args["block_table"][request:request + 1]}
    return c


@pytest.mark.parametrize("dtype", DT)
def test_cu_rows_of_any_values_give_each_request_its_rows(dev, dtype):
    """Request b has the rows from max(cu[b], 0) up to cu[b + 1], max_rows at most: rows of one request are the definition's,
    rows of none, and what lies around out and lse, stay as they are."""
    b = Batch(dev, lengths=[10, 20, 30, 40], nodes=[600, 5, 600, 5], dtype=dtype)
    N, H, D = 1210, b.H, b.D
    for cu in ([0, 1210, 0, 1210, 5000], [0, 600, 300, 1210, 1210], [-7, 2 ** 30, -2 ** 31, 2 ** 31 - 1, 0], [1210, 5, 4, 3, 2],
               [0, 300, 301, 900, 2 ** 31 - 1], [-2 ** 31, 1, 1, 700, 1209]):
        b.args["cu_nodes"].copy_(torch.tensor(cu))
        for most in (600, 300):
            held = torch.full((N + 20, H, D), 9.0, dtype=dtype, device=dev)
            held_lse = torch.full((N + 20, H), 7.0, device=dev)
            b.run(out=held[10:N + 10], lse=held_lse[10:N + 10], max_rows=most)
            out, lse = held[10:N + 10], held_lse[10:N + 10]
            owners = torch.zeros(N, dtype=torch.int64)
            mine = []
            for r in range(4):
                lo = max(cu[r], 0)
                n = max(min(min(max(cu[r + 1], 0), N) - lo, most), 0)
                mine.append((lo, n))
                owners[lo:lo + n] += 1
            none = torch.cat([torch.ones(10, dtype=torch.bool), owners == 0, torch.ones(10, dtype=torch.bool)]).to(dev)
            assert bool((held[none] == 9).all()) and bool((held_lse[none] == 7).all())
            assert bool(torch.isfinite(held).all()) and not bool((lse[(owners > 0).to(dev)] == 7).all(1).any())
            for r, (lo, n) in enumerate(mine):
                alone = (owners[lo:lo + n] == 1).to(dev)
                if n and bool(alone.any()):
                    c = part_of(b, r, lo, n)
                    check(c, out[lo:lo + n][alone], lse[lo:lo + n][alone], [x[alone] for x in c.exact()])


@pytest.mark.parametrize("dtype", DT)
def test_means_of_huge_scores(dev, dtype):
    """As test_huge_scores, V in [1, 2]: out is no less than 1 and no more than 2 but for the weights' and out's roundings, and
    lse is the float64 one within the bound above."""
    b = Batch(dev, lengths=[700], nodes=[600], seed=3, dtype=dtype)
    for t in (b.args["q"], b.args["k_pool"]):
        t.mul_(2.0 ** 13).clamp_(-60000, 60000)
    v = b.args["v_pool"]
    v.copy_(1 + (v.abs() / v.abs().max()).clamp(max=1))
    up = -8 if dtype == F16 else -3
    out, lse = b.run(scale=2.0 ** up)
    c = part_of(b, 0, 0, 600)
    c.args["q"] = c.args["q"].float() * 2.0 ** up * 8  # the default scale is 1 / 8
    _, z, _, dots = c.exact()
    err = 2 * HALF[dtype] + 8000 * U
    assert float(out.min()) >= 1 - err and float(out.max()) <= 2 * (1 + err)
    assert bool(((lse.double() - z).abs() <= (64 + 6) * U * dots + (1300 + 8) * U + 4 * U * z.abs()).all())


@pytest.mark.parametrize("dtype", DT)
def test_queries_of_any_strides(dev, dtype):
    b = Batch(dev, lengths=[77, 0], nodes=[520, 9], dtype=dtype, seed=7)
    want, q = b.run(), b.args["q"]
    pad = torch.nn.functional.pad
    for form in (q.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([q, q], 2)[..., :64], pad(q, (1, 5))[..., 1:65],
                 pad(q, (8, 8))[..., 8:72], q.repeat_interleave(2, 2)[..., ::2], q.repeat_interleave(2, 1)[:, ::2]):
        assert torch.equal(form, q) and form.stride() != q.stride()
        got = b.run(q=form)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_more_units_than_the_plan_keeps(dev):
    """fp32 has units of 32 rows; from 8192 units on the plan works the first ones out anew."""
    rows = [3000, 1, 2601, 0, 1000]
    b = Batch(dev, lengths=[40, 500, 0, 9, 300], nodes=rows, H=40, Hk=1, D=64, dtype=F32, seed=11)
    assert sum(-(-n * 40 // 32) for n in rows) > 8192
    check(b, *b.run(), b.exact())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,most", [(60, 24), (4200, 3)])
def test_short_chunks_padded_replayed_and_on_two_streams(dev, dtype, B, most):
    """Batches that the tree kernels take: one graph for changing lengths and rows, padding rows left as they are, two calls at
    once."""
    lengths, rows = [(k * 31) % 90 for k in range(B)], [(k * 7) % (most + 1) for k in range(B)]
    b = Batch(dev, lengths=lengths, nodes=rows, dtype=dtype, seed=B)
    a, N = b.args, sum(rows)
    pad = {**a, "q": torch.cat([a["q"], a["q"][:20]])}
    b.args = pad
    held = torch.full((N + 20, b.H, b.D), 9.0, dtype=dtype, device=dev)
    held_lse = torch.full((N + 20, b.H), 7.0, device=dev)
    b.run(max_rows=most)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(max_rows=most, out=held, lse=held_lse)
    for turn in range(3):
        b.lengths = [(c + 13 * turn) % 90 for c in lengths]
        b.nodes = rows[turn:] + rows[:turn]
        a["lengths"].copy_(torch.tensor(b.lengths))
        a["cu_nodes"].copy_(torch.tensor([0] + b.nodes).cumsum(0))
        graph.replay()
        eager = b.run(max_rows=most)
        assert torch.equal(held[:N], eager[0][:N]) and torch.equal(held_lse[:N], eager[1][:N])
        assert bool((held[N:] == 9).all()) and bool((held_lse[N:] == 7).all())
        if turn != 1:
            check(b, held[:N], held_lse[:N], b.exact())
    other = Batch(dev, lengths=[9] * 40, nodes=[7] * 40, dtype=dtype, seed=1)
    want = [b.run(max_rows=most), other.run()]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [x.run(stream=t, max_rows=most if x is b else 7) for x, t in zip((b, other), s)]
    torch.cuda.synchronize()
    for g, w, n in zip(got, want, (N, 280)):
        assert torch.equal(g[0][:n], w[0][:n]) and torch.equal(g[1][:n], w[1][:n])
