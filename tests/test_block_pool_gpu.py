"""Block tables, rows to slots, ancestor masks and accepted paths on the GPU:
whole numbers and copied rows, equal to a step-by-step restatement."""
from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------- block tables

def _state(rng, B, W, owned, spare, extra=3):
    """A table whose requests own ``owned[b]`` blocks, and a free list of ``spare``."""
    ids = list(range(sum(owned) + spare))
    rng.shuffle(ids)
    table = [[-1] * W for _ in range(B)]
    for b, k in enumerate(owned):
        table[b][:k] = [ids.pop() for _ in range(k)]
    return table, list(owned), ids + [-7] * (sum(owned) + extra), len(ids)


def _check_update(dev, state, lengths, first, bs, max_rows):
    import halo_amd
    table, owned, free, n_free = state
    dt, dn, df, dc = _i32(table, dev), _i32(owned, dev), _i32(free, dev), _i32([n_free], dev)
    up = halo_amd.update_block_tables(dt, dn, df, dc, _i32(lengths, dev), _i32(first, dev), block_size=bs,
                                      max_rows=max_rows)
    want = paged.update_block_tables(table, owned, free, n_free, lengths, first, block_size=bs, max_rows=max_rows)
    assert dn.tolist() == want[1]
    assert dt.tolist() == want[0]
    assert dc.tolist() == [want[3]]
    assert df.tolist() == want[2]
    assert up.cu_rows.tolist() == want[4]
    assert up.slots.tolist() == want[5]
    assert up.ok.tolist() == want[6]
    return want


@pytest.mark.parametrize("B,bs,seed", [(1, 16, 0), (3, 1, 1), (17, 24, 2), (64, 16, 3), (257, 16, 4), (1024, 32, 5),
                                       (1025, 8, 6), (2300, 16, 7)])
def test_update_grows_shrinks_and_numbers(dev, B, bs, seed):
    rng = random.Random(seed)
    W = 9
    owned = [rng.randint(0, W) for _ in range(B)]
    lengths = [rng.choice([0, 1, rng.randint(0, W * bs), W * bs]) for _ in range(B)]
    first = [rng.randint(0, x) for x in lengths]
    rows = sum(x - f for x, f in zip(lengths, first))
    _check_update(dev, _state(rng, B, W, owned, B * W), lengths, first, bs, rows + 5)


def test_update_of_long_rows_takes_the_wide_slot_launch(dev):
    rng = random.Random(8)
    _check_update(dev, _state(rng, 3, 700, [5, 0, 300], 1200), [11000, 9000, 20], [80, 0, 0], 16, 20000)


@pytest.mark.parametrize("B,W,part", [(90, 200, 0.7), (700, 40, 0.4), (1100, 30, 1.0)])
def test_update_of_thousands_of_blocks(dev, B, W, part):
    """More blocks than one step of the kernel moves, given back past the end of the free list and taken
    until the list is empty."""
    rng = random.Random(B)
    owned = [rng.choice([0, 1, W, rng.randint(0, W)]) for _ in range(B)]
    table, owned, free, n_free = _state(rng, B, W, owned, int(part * sum(owned) / 4))
    lengths = [4 * rng.choice([0, 1, 2, W, rng.randint(0, W)]) for _ in range(B)]
    _check_update(dev, (table, owned, free[:n_free + int(part * sum(owned) / 3)], n_free), lengths,
                  [max(x - 3, 0) for x in lengths], 4, 4 * B)


@pytest.mark.parametrize("spare", [0, 1, 2, 5, 6, 40])
def test_update_serves_in_order_while_blocks_last(dev, spare):
    rng = random.Random(spare)
    owned = [2, 1, 4, 0, 3, 1]
    lengths = [5 * 4, 1 * 4, 2 * 4, 30 * 4, 4 * 4, 2 * 4]  # the fourth does not fit the table
    want = _check_update(dev, _state(rng, 6, 8, owned, spare), lengths, [1, 0, 3, 0, 15, 7], 4, 200)
    assert want[6][3] is False and want[6][1] is True


def test_update_of_odd_lengths(dev):
    rng = random.Random(9)
    _check_update(dev, _state(rng, 4, 6, [1, 2, 0, 6], 10), [-5, 7, 5000, 0], [-3, 9, 4990, 4], 4, 12)


def test_update_of_the_largest_lengths(dev):
    import halo_amd
    most = 2 ** 31 - 1
    up = halo_amd.update_block_tables(_i32([[-1, -1]] * 3, dev), _i32([0] * 3, dev), _i32([5, 6], dev), _i32([2], dev),
                                      _i32([3, most, most], dev), _i32([0] * 3, dev), block_size=4, max_rows=8)
    assert up.ok.tolist() == [True, False, False]
    assert up.cu_rows.tolist() == [0, 3, most, most]  # counts end at the largest int32
    assert up.slots.tolist() == [24, 25, 26] + [-1] * 5


def test_update_drops_ids_past_the_free_list(dev):
    rng = random.Random(10)
    table, owned, free, n_free = _state(rng, 2, 8, [8, 3], 4)
    _check_update(dev, (table, owned, free[:9], n_free), [4, 0], [0, 0], 4, 4)


def test_update_room_for_fewer_rows_and_none(dev):
    rng = random.Random(11)
    s = _state(rng, 3, 8, [1, 1, 1], 20)
    _check_update(dev, s, [20, 9, 30], [3, 1, 0], 4, 10)
    _check_update(dev, s, [20, 9, 30], [3, 1, 0], 4, 0)


def test_update_there_and_back_restores_the_state(dev):
    rng = random.Random(12)
    owned = [rng.randint(0, 9) for _ in range(40)]
    s = _state(rng, 40, 12, owned, 300)
    more = [x * 8 + rng.randint(0, 24) for x in owned]
    t, n, f, c, *_ = paged.update_block_tables(*s, more, more, block_size=8, max_rows=0)
    back = _check_update(dev, (t, n, f, c), [x * 8 for x in owned], [0] * 40, 8, 0)
    assert back[0] == s[0] and back[1] == s[1] and back[3] == s[3]


def test_update_without_a_free_list(dev):
    """An empty free list: lengths that need no new block are served, the others are not."""
    rng = random.Random(13)
    table, owned, _, _ = _state(rng, 3, 4, [2, 1, 0], 0)
    _check_update(dev, (table, owned, [], 0), [16, 9, 0], [14, 8, 0], 8, 4)


def test_update_repairs_counts_past_the_table(dev):
    import halo_amd
    n = _i32([9, -3], dev)
    t = _i32([[4, 5, 6], [-1, -1, -1]], dev)
    free, n_free = _i32([7, -1, -1, -1], dev), _i32([1], dev)
    up = halo_amd.update_block_tables(t, n, free, n_free, _i32([12, 2], dev), _i32([11, 0], dev), block_size=4, max_rows=3)
    assert n.tolist() == [3, 1] and t.tolist() == [[4, 5, 6], [7, -1, -1]] and n_free.tolist() == [0]
    assert up.slots.tolist() == [27, 28, 29]


def test_update_strided_table(dev):
    import halo_amd
    base = torch.full((3, 10), -1, dtype=torch.int32, device=dev)
    free = torch.arange(30, dtype=torch.int32, device=dev)
    n = torch.zeros(3, dtype=torch.int32, device=dev)
    up = halo_amd.update_block_tables(base[:, 2:6], n, free, _i32([30], dev), _i32([9, 0, 5], dev), _i32([0, 0, 4], dev),
                                      block_size=4, max_rows=16)
    assert base.tolist() == [[-1, -1, 29, 28, 27] + [-1] * 5, [-1] * 10, [-1, -1, 26, 25] + [-1] * 6]
    assert up.slots.tolist() == [29 * 4 + i for i in range(4)] + [28 * 4 + i for i in range(4)] + [27 * 4, 25 * 4] \
        + [-1] * 6


# ---------------------------------------------------------------- rows to slots

def _bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("L,N,H,D,bs", [(0, 1, 8, 128, 16), (0, 203, 8, 128, 16), (0, 77, 1, 64, 24), (3, 40, 2, 64, 7),
                                        (0, 33, 3, 80, 16), (0, 9, 2, 5, 4), (0, 5, 40, 256, 16)])
def test_append_rows(dev, dtype, L, N, H, D, bs):
    import halo_amd
    g = torch.Generator(device=dev).manual_seed(N)
    P = -(-N // bs) + 3
    lead = (L,) if L else ()
    k, v = (torch.randn(lead + (N, H, D), generator=g, device=dev).to(dtype) for _ in range(2))
    kp, vp = (torch.randn(lead + (P, H, bs, D), generator=g, device=dev).to(dtype) for _ in range(2))
    slots = torch.randperm(P * bs, generator=g, device=dev)[:N]
    wk, wv = kp.clone(), vp.clone()
    for i, s in enumerate(slots.tolist()):
        wk[..., s // bs, :, s % bs, :] = k[..., i, :, :]
        wv[..., s // bs, :, s % bs, :] = v[..., i, :, :]
    halo_amd.append_rows(k, v, slots, kp, vp)
    assert torch.equal(_bits(kp), _bits(wk)) and torch.equal(_bits(vp), _bits(wv))


def test_append_skips_slots_outside_the_pool(dev):
    import halo_amd
    k = torch.randn(6, 2, 64, device=dev)
    kp, vp = torch.zeros(3, 2, 4, 64, device=dev), torch.zeros(3, 2, 4, 64, device=dev)
    slots = torch.tensor([-1, 5, 12, -2 ** 63, 2 ** 62, 11], device=dev)
    halo_amd.append_rows(k, k + 1, slots, kp, vp)
    want = torch.zeros_like(kp)
    want[1, :, 1], want[2, :, 3] = k[1], k[5]
    assert torch.equal(kp, want)
    assert torch.equal(vp, torch.where(want != 0, want + 1, 0))


def test_append_strided_rows_and_pools(dev):
    """Rows as slices of a fused projection, pools as every other head of wider ones, an odd start."""
    import halo_amd
    for off in (0, 1):
        qkv = torch.randn(10, 3, 4, 64 + 2 * off, device=dev).to(torch.bfloat16)
        k, v = qkv[:, 1, ::2, off:off + 64], qkv[:, 2, ::2, off:off + 64]
        kw, vw = (torch.zeros(5, 4, 6, 64, device=dev, dtype=torch.bfloat16) for _ in range(2))
        slots = torch.randperm(30, device=dev)[:10]
        halo_amd.append_rows(k, v, slots, kw[:, 1::2], vw[:, 1::2])
        for i, s in enumerate(slots.tolist()):
            assert torch.equal(kw[s // 6, 1::2, s % 6], k[i]) and torch.equal(vw[s // 6, 1::2, s % 6], v[i])
        assert not kw[:, ::2].any() and not vw[:, ::2].any()


def test_append_no_rows(dev):
    import halo_amd
    kp = torch.ones(2, 1, 4, 64, device=dev)
    e = torch.empty(0, 1, 64, device=dev)
    halo_amd.append_rows(e, e, torch.empty(0, dtype=torch.int64, device=dev), kp, kp.clone())
    assert bool((kp == 1).all())


# ---------------------------------------------------------------- ancestor masks

def _tree(rng, n, kind):
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "roots":
        return [-1] * n
    if kind == "odd":
        return [rng.choice([-1, -2 ** 31, i, i + 1, n, 2 ** 31 - 1, rng.randint(0, max(0, i - 1))]) for i in range(n)]
    return [rng.randint(max(-1, i - 9), i - 1) for i in range(n)]


@pytest.mark.parametrize("kind", ["tree", "chain", "roots", "odd"])
@pytest.mark.parametrize("sizes", [[1], [64], [65], [3, 0, 17, 1], [200, 1, 128], [512, 300, 257], [5] * 300])
def test_tree_layout(dev, kind, sizes):
    import halo_amd
    rng = random.Random(len(sizes) + sizes[0])
    trees = [_tree(rng, n, kind) for n in sizes]
    cu = np.concatenate([[0], np.cumsum(sizes)]).tolist()
    W = -(-max(sizes) // 64)
    mask, depth = halo_amd.tree_layout(_i32(sum(trees, []), dev), _i32(cu, dev), max_nodes=max(sizes))
    sets = [s for t in trees for s in paged.ancestors(t)]
    assert np.array_equal(mask.cpu().numpy(), paged.words(sets, W))
    assert depth.tolist() == [len(s) - 1 for s in sets]


def test_tree_layout_leaves_padding_and_further_nodes(dev):
    import halo_amd
    parents = _i32([-1, 0, 1, -1, 0, 1, 2, 3, 9, 9], dev)
    mask = torch.full((10, 1), 77, dtype=torch.int64, device=dev)
    depth = torch.full((10,), 78, dtype=torch.int32, device=dev)
    halo_amd.tree_layout(parents, _i32([0, 3, 8], dev), max_nodes=4, mask=mask, depth=depth)
    assert mask[:, 0].tolist() == [1, 3, 7, 1, 3, 7, 15, 77, 77, 77]
    assert depth.tolist() == [0, 1, 2, 0, 1, 2, 3, 78, 78, 78]


def test_tree_layout_of_any_cu_nodes(dev):
    """Ranges whose difference does not fit 32 bits are empty, or cut at the nodes there are."""
    import halo_amd
    parents = _i32([-1, 0, 1, 0, 2, 9, 9], dev)
    for cu, there in (([-7, 2 ** 30, -2 ** 31, 2 ** 31 - 1, 0], True), ([2 ** 31 - 1, -2 ** 31, 2 ** 30, -5, -1], True),
                      ([7, 4, 3, 2, -2 ** 31], False)):
        mask = torch.full((7, 1), 77, dtype=torch.int64, device=dev)
        depth = torch.full((7,), 78, dtype=torch.int32, device=dev)
        halo_amd.tree_layout(parents, _i32(cu, dev), max_nodes=5, mask=mask, depth=depth)
        assert mask[:, 0].tolist() == ([1, 3, 7, 9, 23] if there else [77] * 5) + [77] * 2
        assert depth.tolist() == ([0, 1, 2, 1, 3] if there else [78] * 5) + [78] * 2


# ---------------------------------------------------------------- accepted paths

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L,B,H,D,bs,P,n", [(1, 1, 8, 128, 16, 5, 12), (4, 3, 2, 64, 7, 9, 40), (2, 5, 3, 80, 24, 64, 200),
                                            (1, 2, 1, 5, 4, 1, 3)])
def test_commit_path(dev, dtype, L, B, H, D, bs, P, n):
    import halo_amd
    rng = random.Random(B * P)
    lengths = [rng.choice([0, rng.randint(1, 50)]) for _ in range(B)]
    W = -(-(max(lengths) + n) // bs)
    ids = list(range(B * W + 2))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(W)] for _ in range(B)]
    path = [sorted(rng.sample(range(n), P)) for _ in range(B)]  # moves that read rows other moves write among them
    n_path = [rng.randint(0, P) for _ in range(B)]
    g = torch.Generator(device=dev).manual_seed(P)
    shape = ((L,) if L > 1 else ()) + (B * W + 2, H, bs, D)
    kp, vp = (torch.randn(shape, generator=g, device=dev).to(dtype) for _ in range(2))
    wk, wv = kp.clone(), vp.clone()
    for b in range(B):
        for j in range(n_path[b]):
            s, d = lengths[b] + path[b][j], lengths[b] + j
            for w, p in ((wk, kp), (wv, vp)):
                w[..., table[b][d // bs], :, d % bs, :] = p[..., table[b][s // bs], :, s % bs, :]
    new = halo_amd.commit_path(kp, vp, _i32(table, dev), _i32(lengths, dev), _i32(path, dev), _i32(n_path, dev))
    assert new.tolist() == [a + b for a, b in zip(lengths, n_path)]
    assert torch.equal(_bits(kp), _bits(wk)) and torch.equal(_bits(vp), _bits(wv))


def test_commit_path_ends_where_it_does_not_rise_or_leaves_the_table(dev):
    import halo_amd
    kp = torch.arange(12 * 4, device=dev, dtype=torch.float32).view(12, 1, 4, 1).expand(12, 1, 4, 64).contiguous()
    vp = kp + 1000
    table = _i32([[0, 1], [2, 3], [4, 5], [6, -1], [8, 99], [10, 11]], dev)
    lengths = _i32([2, 2, 2, 2, 2, -4], dev)
    path = _i32([[1, 3, 3, 5], [0, -1, 2, 3], [2, 5, 6, 7], [1, 2, 3, 4], [0, 1, 3, 4], [1, 2, 3, 7]], dev)
    n_path = _i32([4, 4, 4, 4, 99, 4], dev)
    got = halo_amd.commit_path(kp, vp, table, lengths, path, n_path)
    assert got.tolist() == [4, 3, 4, 3, 4, 4]
    rows = kp[:, 0, :, 0].reshape(-1)
    want = torch.arange(48, device=dev, dtype=torch.float32)
    want[2], want[3] = 3, 5                        # rows 2 + {1, 3} of the first
    want[16 + 2], want[16 + 3] = 16 + 4, 16 + 7    # third: {2, 5}; 6 and 7 lie past its two blocks
    want[24 + 2] = 24 + 3                          # fourth: row 2 + 2 is in a block that is not there
    want[40:44] = torch.tensor([41., 42., 43., 47.], device=dev)
    assert torch.equal(rows, want)
    assert torch.equal(vp[:, 0, :, 5].reshape(-1), want + 1000)


def test_pool_of_the_block_store(dev):
    from halo_amd import TieredStorage, append_rows
    st = TieredStorage(tiers=["gpu", "dram"], num_layers=2, num_kv_heads=2, head_dim=64, block_size=4,
                       dtype=torch.float16, device=dev, max_blocks=6)
    k = torch.randn(2, 5, 2, 64, device=dev).half()
    append_rows(k, -k, torch.arange(9, 14, device=dev), *st.pool())
    kb, vb = st.read_block(layer=1, block=2)
    assert torch.equal(kb[:, 1:4], k[1, :3].transpose(0, 1)) and torch.equal(vb[:, 1:4], -k[1, :3].transpose(0, 1))
    assert st.pool("gpu", 1)[0].data_ptr() == st.pool()[0][1].data_ptr()
