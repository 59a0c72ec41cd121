"""How a call of tree attention is cut into items, restated from the lengths:
the launch's shape, the share of tiles that a workgroup finds on the device (its
float sums in their order) and the items' tiles."""
from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

F = np.float32


class Shape(NamedTuple):
    nw: int         # 32-row waves of a unit; 1: the narrow kernels
    kt: int         # keys of a tile
    slots: int
    min_tiles: int
    units: int      # at most
    grid: int
    merge_units: int
    partials: int   # of 32 rows, at most
    ws_bytes: int


def shape(dtype, B, H, Hk, D, max_rows, max_nodes) -> Shape:
    f32 = dtype == torch.float32
    rows = max_nodes * (H // Hk)
    nw = 1 if f32 or rows <= 32 else 2 if rows <= 64 else 4 if rows <= 128 else 8
    kt = 32 if nw == 1 else 64
    units = B * Hk * -(-rows // (32 * nw))
    few = nw == 1 and units <= 32
    slots = 256 if few or nw == 8 or (f32 and D == 128) else 512
    min_tiles = 4 if nw == 1 else 2
    merge = -(-(max_rows + max_nodes) // kt) > min_tiles
    grid = max(slots // 2 + units, slots) if merge else units
    partials = slots * nw if merge else 0
    return Shape(nw, kt, slots, min_tiles, units, grid, min(units, slots // 2), partials, partials * (32 * D * 4 + 32 * 8))


def _wave_sums(x):
    """Sums over 64 lanes (last axis) in the order of the device's scan."""
    x = x.reshape(x.shape[0], 4, 16).copy()
    for s in (1, 2, 4, 8):
        y = np.zeros_like(x)
        y[..., s:] = x[..., :-s]
        x = x + y
    x[:, 1], x[:, 3] = x[:, 1] + x[:, 0, 15:], x[:, 3] + x[:, 2, 15:]
    return x[:, 3, 15] + x[:, 1, 15]


def share(s: Shape, tiles, units) -> int:
    """L, the longest item: ``tiles`` and ``units`` of each request."""
    B = len(tiles)
    each = 1 if B <= 64 else 4
    pad = -B % (64 * each)
    t = np.concatenate([units, np.zeros(pad, int)]).astype(F) * np.concatenate([tiles, np.zeros(pad, int)]).astype(F)
    t = t.reshape(-1, 64, each)
    lane = t[..., 0]
    for k in range(1, each):
        lane = lane + t[..., k]
    total = np.cumsum(_wave_sums(lane), dtype=F)[-1]
    n = int(units.sum())
    room = s.slots - n if s.slots > 2 * n else s.slots // 2
    x = int(min(np.ceil(F(total * F(1 + 2.0 ** -14)) / F(room)), F(1e9)))
    even = 4 if s.nw == 1 else 1
    return max(-(-x // even) * even, s.min_tiles)


class Cuts(NamedTuple):
    shape: Shape
    L: int
    items: int
    cut_units: int
    partials: int      # of 32 rows
    sizes: list        # of the items' (first tile, tiles, first tile with tree rows), one head and row block of each request


def cuts(dtype, H, Hk, D, max_rows, max_nodes, lengths, nodes, sizes=True) -> Cuts:
    lengths, nodes = np.minimum(np.asarray(lengths), max_rows), np.minimum(np.asarray(nodes), max_nodes)
    s = shape(dtype, len(lengths), H, Hk, D, max_rows, max_nodes)
    tiles = np.where(nodes > 0, -(-(lengths + nodes) // s.kt), 0)
    units = Hk * -(-nodes * (H // Hk) // (32 * s.nw))
    L = share(s, tiles, units)
    n = -(-tiles // L)
    many = n > 1
    got = []
    if sizes:
        for c, t, k in zip(lengths.tolist(), tiles.tolist(), n.tolist()):
            got += [(t * i // k, t * (i + 1) // k - t * i // k, c // s.kt) for i in range(k)]
    return Cuts(s, L, int((units * n).sum()), int(units[many].sum()), int((units * n)[many].sum()) * s.nw, got)


class Batch:
    """Requests over a pool whose blocks they share in any order: many rows attended, few rows held."""

    def __init__(self, dev, *, lengths, nodes, H, Hk, D, bs, dtype, seed, blocks=300, holes=0.0, masks=True):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.H, self.Hk, self.D, self.bs = dtype, H, Hk, D, bs
        self.lengths, self.nodes = list(lengths), list(nodes)
        W = max(-(-(c + n) // bs) for c, n in zip(lengths, nodes)) + 1
        table = rng.integers(0, blocks, (len(lengths), W))
        if holes:  # in front of the tree rows, which nodes shall see
            cols = np.arange(W)[None] < np.asarray(lengths)[:, None] // bs
            table = np.where(cols & (rng.random(table.shape) < holes), rng.choice([-1, blocks, 2 ** 31 - 1]), table)
        N = sum(nodes)
        self.max_nodes, self.W = max(nodes), W
        words = -(-self.max_nodes // 64)
        bits = rng.integers(-2 ** 63, 2 ** 63, (N, words), dtype=np.int64)
        self.args = dict(q=torch.randn(N, H, D, generator=g).to(dtype), k_pool=torch.randn(blocks, Hk, bs, D, generator=g).to(dtype),
                         v_pool=torch.randn(blocks, Hk, bs, D, generator=g).to(dtype),
                         block_table=torch.from_numpy(table).int(), lengths=torch.tensor(self.lengths, dtype=torch.int32),
                         cu_nodes=torch.tensor(np.concatenate([[0], np.cumsum(nodes)]), dtype=torch.int32),
                         mask=torch.from_numpy(bits) if masks else None)
        self.args = {k: t if t is None else t.to(dev) for k, t in self.args.items()}

    def cuts(self) -> Cuts:
        return cuts(self.dtype, self.H, self.Hk, self.D, self.W * self.bs, self.max_nodes, self.lengths, self.nodes)

    def run(self, **kw):
        import halo_amd
        return halo_amd.tree_attention(**self.args, max_nodes=self.max_nodes, return_lse=True, **kw)

    def exact(self, only=None):
        """out, lse, the weighted mean of |v| and the largest scale * sum |q_d k_d| in float64 (of the requests ``only``)."""
        a, rep = self.args, self.H // self.Hk
        dev = a["q"].device
        got = []
        at = np.concatenate([[0], np.cumsum(self.nodes)])
        for b in range(len(self.lengths)) if only is None else only:
            c, n = self.lengths[b], self.nodes[b]
            pos = torch.arange(c + n, device=dev)
            blk = a["block_table"][b].long()[pos // self.bs]
            there = (blk >= 0) & (blk < a["k_pool"].shape[0])
            blk = torch.where(there, blk, 0)
            k, v = (a[p][blk, :, pos % self.bs].double() for p in ("k_pool", "v_pool"))  # (T, Hk, D)
            j = torch.arange(n, device=dev)
            if a["mask"] is None:
                tree = j[None] <= j[:, None]
            else:
                tree = (a["mask"][at[b]:at[b + 1]][:, j // 64] >> (j % 64)) & 1 == 1
            sees = there & torch.cat([torch.ones(n, c, dtype=torch.bool, device=dev), tree], 1)
            q = a["q"][at[b]:at[b + 1]].double()
            per = []
            for h in range(self.H):
                kh, vh = k[:, h // rep].contiguous(), v[:, h // rep].contiguous()
                kt = kh.T.contiguous()
                s = (q[:, h].contiguous() @ kt * self.D ** -0.5).masked_fill(~sees, -torch.inf)
                z = torch.logsumexp(s, 1)
                w = torch.exp(s - torch.where(z == -torch.inf, 0, z)[:, None])
                dots = (q[:, h].abs().contiguous() @ kt.abs() * self.D ** -0.5).masked_fill(~sees, 0).amax(1)
                per.append((w @ vh, z, w @ vh.abs(), dots))
            got.append([torch.stack(x, 1) for x in zip(*per)])
        return [torch.cat(x) for x in zip(*got)]
