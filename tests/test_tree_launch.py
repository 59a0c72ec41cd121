"""Tree attention's cut of a batch into items, on the host: what it launches and
the room of its partials hold for every batch."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import tree_launch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype,code", [(F32, 0), (BF16, 1), (F16, 2)])
@pytest.mark.parametrize("B,H,Hk,D,rows,nodes", [(1, 8, 8, 64, 128, 1), (1, 8, 8, 64, 1000, 1), (4, 32, 8, 128, 5000, 8),
                                                 (5, 32, 8, 128, 5000, 8), (16, 28, 4, 128, 32768, 12),
                                                 (1, 32, 8, 128, 32768, 64), (300, 4, 1, 64, 90, 16), (2, 64, 1, 128, 9000, 512)])
def test_workspace_is_that_of_the_restated_shape(dtype, code, B, H, Hk, D, rows, nodes):
    from halo_amd import _native as nat
    if not nat.loadable():
        pytest.skip("library not built (run __graft_entry__.build())")
    s = tree_launch.shape(dtype, B, H, Hk, D, rows, nodes)
    assert nat._load().halo_tree_workspace_size(code, B, H, Hk, D, rows, nodes) == s.ws_bytes


def _batches(rng, B):
    """Lengths that could lead the float sum of tiles astray: any, and few long requests before, between and behind short ones."""
    yield np.exp(rng.uniform(0, np.log(2e6), B)).astype(int)
    for long in (3e4, 3e7):
        n = np.ones(B, int)
        n[:min(B, 300)] = int(long) + rng.integers(0, 64, min(B, 300))
        yield n
        yield n[::-1].copy()
        yield rng.permutation(n)
    yield np.full(B, 100003)


@pytest.mark.parametrize("B", [1, 2, 7, 40, 64, 65, 256, 300, 1025, 5000, 1 << 18, 1 << 20])
@pytest.mark.parametrize("dtype,H,Hk,D,nodes", [(BF16, 4, 1, 128, 1), (F16, 8, 2, 64, 12), (BF16, 8, 1, 64, 20), (F32, 2, 1, 128, 33)])
def test_items_and_partials_fit_every_batch(B, dtype, H, Hk, D, nodes):
    rng = np.random.default_rng(B)
    for lengths in _batches(rng, B):
        n = rng.integers(0, nodes + 1, B)
        c = tree_launch.cuts(dtype, H, Hk, D, 1 << 25, nodes, lengths, n, sizes=False)
        assert c.items <= c.shape.grid and c.cut_units <= c.shape.merge_units and c.partials <= c.shape.partials


@pytest.mark.parametrize("masks", [True, False])
def test_the_batch_reference_is_the_definition(masks):
    from oracle import paged
    b = tree_launch.Batch("cpu", lengths=[40, 0, 7], nodes=[5, 70, 1], H=4, Hk=2, D=64, bs=8, dtype=F32, seed=1, blocks=9,
                          holes=0.2, masks=masks)
    a = b.args
    sees = []
    for n, at in zip(b.nodes, a["cu_nodes"].tolist()):
        for i in range(n):
            sees.append({j for j in range(n) if (j <= i if not masks else int(a["mask"][at + i, j // 64]) >> (j % 64) & 1)})
    want = paged.attend(*[a[k].double().numpy() for k in ("q", "k_pool", "v_pool")], a["block_table"].tolist(), b.lengths,
                        a["cu_nodes"].tolist(), sees, 64 ** -0.5)
    for x, y in zip(b.exact(), want):
        np.testing.assert_allclose(x.numpy(), y, rtol=1e-12, atol=1e-13)
