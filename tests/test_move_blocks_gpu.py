"""Forked, given up and compacted blocks on the GPU, against the definition."""
from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle import serving

pytestmark = pytest.mark.gpu
I32 = torch.int32
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Store:
    """Requests over a pool, with the same state in lists and arrays."""

    def __init__(self, dev, *, B, W, P, bs=16, L=2, H=2, D=64, dtype=BF16, seed=0, cap=None, wide=0):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.bs, self.rng = dev, bs, random.Random(seed)
        shape = (P, H, bs, D) if L == 0 else (L, P, H, bs, D)
        self.kp, self.vp = (torch.randn(shape, generator=g).to(dtype).to(dev) for _ in range(2))
        free = list(range(P))
        self.rng.shuffle(free)
        cap = P if cap is None else cap
        self.table, self.n = [[-1] * W for _ in range(B)], [0] * B
        self.free, self.n_free = free[:cap], min(cap, P)
        self.shared, self.lengths = [0] * P, [0] * B
        full = torch.full((B, W + wide), -7, dtype=I32, device=dev)
        self.t_table = full[:, :W]
        self.t_table.fill_(-1)
        self.t = [torch.tensor(x, dtype=I32, device=dev) for x in (self.n, self.free, [self.n_free], self.shared, self.lengths)]

    def give(self, b, rows, spare=0):
        """Request b holds this many rows, and spare blocks behind them."""
        need = -(-rows // self.bs) + spare
        while self.n[b] < need:
            self.table[b][self.n[b]] = self.free[self.n_free - 1]
            self.n_free -= 1
            self.n[b] += 1
        self.lengths[b] = rows

    def send(self):
        self.t_table.copy_(torch.tensor(self.table, dtype=I32))
        for t, x in zip(self.t, (self.n, self.free, [self.n_free], self.shared, self.lengths)):
            t.copy_(torch.tensor(x, dtype=I32))

    def pools(self):
        return [(t if t.dim() == 5 else t[None]).double().cpu().numpy().copy() for t in (self.kp, self.vp)]

    def fork(self, source, call=None, **kw):
        import halo_amd
        pools = self.pools()
        n, free, n_free, shared, lengths = self.t
        src = torch.tensor(source, dtype=I32, device=self.dev)
        got = call(src) if call else halo_amd.fork_blocks(self.t_table, n, free, n_free, shared, lengths, src, self.kp, self.vp,
                                                          **kw)
        torch.cuda.synchronize()
        (self.table, self.n, self.free, self.n_free, self.shared, self.lengths, ok) = serving.fork(
            self.table, self.n, self.free, self.n_free, self.shared, self.lengths, source, self.bs, pools)
        assert got[0].dtype == I32 and got[1].dtype == torch.bool and got[1].tolist() == [ok]
        assert got[0].tolist() == self.lengths
        lengths.copy_(got[0])
        self.same(pools)
        return ok

    def compact(self, call=None, **kw):
        import halo_amd
        pools = self.pools()
        n, free, n_free, shared, _ = self.t
        got = call() if call else halo_amd.compact_blocks(self.t_table, n, free, n_free, shared, self.kp, self.vp, **kw)
        torch.cuda.synchronize()
        self.table, self.free, self.n_free, self.shared, new_id, n_used = serving.compact(
            self.table, self.n, self.free, self.n_free, self.shared, pools)
        assert got[0].dtype == got[1].dtype == I32 and got[0].tolist() == new_id and got[1].tolist() == [n_used]
        self.same(pools)

    def same(self, pools):
        assert self.t_table.tolist() == self.table
        for t, x in zip(self.t, (self.n, self.free, [self.n_free], self.shared)):
            assert t.tolist() == x
        for t, x in zip((self.kp, self.vp), pools):
            assert np.array_equal((t if t.dim() == 5 else t[None]).double().cpu().numpy(), x)


@pytest.mark.parametrize("L,H,D,dtype,bs", [(0, 1, 64, BF16, 16), (1, 2, 128, F16, 8), (3, 4, 64, F32, 24), (2, 3, 5, F16, 3),
                                            (2, 1, 6, BF16, 1), (1, 8, 7, F32, 64)])
def test_beams(dev, L, H, D, dtype, bs):
    """Beams of three requests that grow and are picked, again and again."""
    s = Store(dev, B=12, W=14, P=160, bs=bs, L=L, H=H, D=D, dtype=dtype, seed=D, wide=3)
    for g in range(3):
        s.give(4 * g, [5 * bs + 2, 3 * bs, 1][g], spare=g % 2)
    s.send()
    assert s.fork([b // 4 * 4 for b in range(12)])
    for step in range(6):
        for b in range(12):  # the new token's row, as update_block_tables would give it a block
            s.give(b, s.lengths[b] + 1)
        s.send()
        assert s.fork([b // 4 * 4 + s.rng.randrange(4) for b in range(12)])
    assert s.fork([-1] * 12)
    assert sorted(s.free[:s.n_free]) == list(range(160)) and not any(s.shared)


@pytest.mark.parametrize("seed", range(8))
def test_any_sources(dev, seed):
    rng = random.Random(seed)
    B = rng.choice([1, 2, 7, 40])
    bs = rng.choice([1, 4, 16])
    s = Store(dev, B=B, W=9, P=9 * B + 7, bs=bs, L=rng.randint(1, 3), H=2, D=rng.choice([8, 5]), dtype=F32, seed=seed)
    for b in range(B):
        if rng.random() < 0.7:
            s.give(b, rng.randint(0, 7 * bs), spare=rng.randint(0, 2))
    s.send()
    for step in range(5):
        s.fork([rng.choice([-5, -1, B, 2 ** 31 - 1, b, b, rng.randrange(B), rng.randrange(B), 0]) for b in range(B)])
        for b in range(B):
            if rng.random() < 0.5 and s.n_free > 3 and s.lengths[b] < 7 * bs:
                s.give(b, s.lengths[b] + rng.randint(0, bs))
        s.send()


def test_free_list_that_does_not_cover_the_copies(dev):
    s = Store(dev, B=6, W=4, P=7, bs=4, seed=1)
    s.give(0, 6)
    s.give(1, 9)
    s.send()
    assert s.n_free == 2
    assert not s.fork([0, 1, 0, 0, 1, -1])   # three copies, two free blocks
    assert s.fork([0, 1, 0, 1, -1, -1])      # two
    assert s.n_free == 0
    assert not s.fork([0, 1, 2, 3, 0, -1])
    assert s.fork([-1, 1, 2, 3, 2, -1])      # the block that row 0 gives up is enough
    assert s.fork([-1] * 6) and s.n_free == 7


def test_lengths_beyond_the_blocks_and_below_zero(dev):
    s = Store(dev, B=4, W=5, P=20, bs=8, seed=3)
    s.give(0, 20)
    s.give(1, 16)
    s.lengths[0], s.lengths[1], s.lengths[2] = 500, -3, 9
    s.send()
    assert s.fork([0, 0, 1, 2])


def test_a_short_free_buffer_drops_ids(dev):
    s = Store(dev, B=5, W=6, P=30, bs=4, seed=4)
    for b in range(5):
        s.give(b, 18)
    s.free, s.n_free = s.free[:7], min(s.n_free, 4)
    s.t[1] = torch.zeros(7, dtype=I32, device=dev)
    s.send()
    assert s.fork([-1, 1, 1, -1, 4])


def test_entries_that_are_no_blocks(dev):
    """-1 and ids past the pool among a row's blocks are handed on, and neither counted, freed nor copied."""
    s = Store(dev, B=4, W=5, P=20, bs=4, seed=5)
    s.give(0, 16)
    s.table[0][1], s.table[0][2] = -1, 77
    s.send()
    assert s.fork([0, 0, 0, -1])
    assert s.fork([-1, 1, 1, -1])


@pytest.mark.parametrize("B,P", [(300, 1200), (4096, 9000)])
def test_many_requests(dev, B, P):
    s = Store(dev, B=B, W=3, P=P, bs=2, L=1, H=1, D=4, dtype=F32, seed=B)
    for b in range(0, B, 3):
        s.give(b, s.rng.randint(0, 4))
    s.send()
    assert s.fork([b - b % 3 if s.rng.random() < 0.8 else -1 for b in range(B)])
    assert s.fork([s.rng.randrange(-1, B) for b in range(B)])


@pytest.mark.parametrize("L,H,D,dtype,bs", [(0, 1, 64, BF16, 16), (1, 2, 128, F16, 8), (3, 4, 64, F32, 24), (2, 3, 5, F16, 3),
                                            (2, 1, 6, BF16, 1)])
def test_compaction(dev, L, H, D, dtype, bs):
    s = Store(dev, B=6, W=7, P=60, bs=bs, L=L, H=H, D=D, dtype=dtype, seed=D, wide=1)
    for b in range(4):
        s.give(b, (b + 1) * bs + b % 2)
    s.send()
    assert s.fork([0, 1, 1, 3, 3, 0])
    s.compact()
    used = {x for row, n in zip(s.table, s.n) for x in row[:n]}
    assert used == set(range(len(used)))
    s.compact()  # nothing is left to move
    assert s.fork([-1, 1, -1, 3, 4, -1])
    s.compact()
    assert s.fork([1, 1, 4, 3, 4, -1])


@pytest.mark.parametrize("seed", range(6))
def test_compaction_of_any_pool(dev, seed):
    """Blocks that are neither in a table nor free stay; empty and full pools; one block."""
    rng = random.Random(seed)
    B, P = rng.choice([1, 3, 20]), rng.choice([1, 5, 64, 3000])
    s = Store(dev, B=B, W=max(2, min(P // B, 40)), P=P, bs=2, L=2, H=1, D=4, dtype=F32, seed=seed)
    foreign = rng.randint(0, s.n_free // 3)
    s.n_free -= foreign
    for b in range(B):
        if s.n_free and rng.random() < 0.9:
            s.give(b, min(rng.randint(0, 80), 2 * len(s.table[b]), 2 * s.n_free))
    keep = rng.choice([0, s.n_free, s.n_free // 2])
    s.free[:keep] = s.free[s.n_free - keep:s.n_free]
    s.n_free = keep
    s.send()
    s.compact()


def test_compaction_with_entries_that_are_no_blocks(dev):
    s = Store(dev, B=3, W=5, P=20, bs=4, seed=5)
    s.give(0, 16)
    s.give(2, 9)
    s.table[0][1], s.table[0][2] = -1, 77
    s.free[0], s.free[1] = -3, 20
    s.send()
    # ids that are none leave the free list, and so does the room that they had
    s.compact()


def test_forks_replayed(dev):
    import halo_amd
    s = Store(dev, B=8, W=6, P=80, bs=8, seed=6)
    s.give(0, 27)
    s.give(4, 33)
    s.send()
    assert s.fork([0, 0, 0, 0, 4, 4, 4, 4])
    src = torch.zeros(8, dtype=I32, device=dev)
    n, free, n_free, shared, lengths = s.t
    keep = [x.clone() for x in (s.t_table, n, free, n_free, shared, s.kp, s.vp)]
    graph = torch.cuda.CUDAGraph()
    src.copy_(torch.arange(8, dtype=I32))
    with torch.cuda.graph(graph):
        got = halo_amd.fork_blocks(s.t_table, n, free, n_free, shared, lengths, src, s.kp, s.vp)
    for x, y in zip((s.t_table, n, free, n_free, shared, s.kp, s.vp), keep):
        assert torch.equal(x, y)  # capturing runs nothing

    def call(source):
        src.copy_(source)
        graph.replay()
        return got
    for _ in range(5):
        assert s.fork([b // 4 * 4 + s.rng.randrange(4) for b in range(8)], call=call)
        assert s.fork([b // 4 * 4 + s.rng.randrange(4) for b in range(8)])
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        moved = halo_amd.compact_blocks(s.t_table, n, free, n_free, shared, s.kp, s.vp)

    def compact():
        graph2.replay()
        return moved
    for _ in range(3):
        s.compact(call=compact)
        assert s.fork([b // 4 * 4 + s.rng.randrange(4) for b in range(8)])


def test_another_stream(dev):
    s = Store(dev, B=6, W=6, P=50, bs=8, seed=7)
    s.give(0, 27)
    s.give(3, 13)
    s.send()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert s.fork([0, 0, 0, 3, 3, -1], stream=side)
    s.compact(stream=side)


def test_pools_past_32_bit_offsets(dev):
    """Blocks beyond 2^32 bytes of a pool, copied and moved."""
    import halo_amd
    P, D, bs = 2 ** 32 // (2 * 64 * 128) + 100, 128, 64
    kp = torch.zeros((P, 1, bs, D), dtype=BF16, device=dev)
    vp = torch.zeros_like(kp)
    i32 = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    table, n, lengths = i32([[P - 2, -1], [-1, -1]]), i32([1, 0]), i32([40, 0])
    free, n_free, shared = i32([5, P - 1]), i32([2]), torch.zeros(P, dtype=I32, device=dev)
    kp[P - 2], vp[P - 2] = 3, 4
    new, ok = halo_amd.fork_blocks(table, n, free, n_free, shared, lengths, i32([0, 0]), kp, vp)
    assert ok.tolist() == [True] and table.tolist() == [[P - 2, -1], [P - 1, -1]] and new.tolist() == [40, 40]
    assert bool((kp[P - 1, 0, :40] == 3).all()) and not bool(kp[P - 1, 0, 40:].any()) and bool((vp[P - 1, 0, :40] == 4).all())
    new_id, used = halo_amd.compact_blocks(table, n, free, n_free, shared, kp, vp)
    assert used.tolist() == [2] and table.tolist() == [[P - 2, -1], [5, -1]] and new_id[P - 1].item() == 5
    assert bool((kp[5, 0, :40] == 3).all()) and bool((vp[5, 0, :40] == 4).all()) and free[:1].tolist() == [P - 1]


@pytest.mark.parametrize("B,W,P", [(10, 1700, 900), (3, 5, 9000), (600, 4, 2000)])
def test_tables_and_pools_that_one_workgroup_does_not_hold(dev, B, W, P):
    """More entries, blocks or requests than the single launch takes."""
    s = Store(dev, B=B, W=W, P=P, bs=4, L=2, H=1, D=8, dtype=F32, seed=B)
    for b in range(0, B, 2):
        s.give(b, s.rng.randint(0, 4 * min(W, P // B) - 4))
    s.send()
    s.compact()
    for step in range(4):
        s.fork([s.rng.choice([-1, b, b, s.rng.randrange(B), s.rng.randrange(B)]) for b in range(B)])
        for b in range(B):
            if s.rng.random() < 0.5 and s.n_free > 3 and s.lengths[b] < 4 * W - 4:
                s.give(b, s.lengths[b] + s.rng.randint(0, 4))
        s.send()
    s.compact()


@pytest.mark.parametrize("B,W,P", [(4, 7, 33000), (33, 2000, 3000)])
def test_compaction_beyond_one_workgroup(dev, B, W, P):
    s = Store(dev, B=B, W=W, P=P, bs=1, L=1, H=1, D=4, dtype=F32, seed=W)
    for b in range(B):
        s.give(b, s.rng.randint(0, min(W, P // B // 2)))
    s.n_free -= 11  # blocks of somebody else
    s.send()
    s.compact()
    assert s.fork([b if b % 3 else -1 for b in range(B)])
    s.compact()
