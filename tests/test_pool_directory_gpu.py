"""Rows written to the GPU tier's pool and the store's directory: what is read,
and what a move back brings, after blocks were moved out."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
L, H, BS, D, BLOCKS = 3, 2, 4, 64, 8


@pytest.fixture
def store(dev):
    from halo_amd import TieredStorage
    st = TieredStorage(tiers=["gpu", "dram"], num_layers=L, num_kv_heads=H, head_dim=D, block_size=BS,
                       dtype=torch.bfloat16, device=dev, max_blocks=BLOCKS)
    for layer in range(L):
        for b in range(BLOCKS):
            st.write_new_block(layer=layer, block=b, keys=torch.full((H, BS, D), float(b), device=dev),
                               values=torch.full((H, BS, D), 100.0 + b, device=dev))
        st.move_blocks(layer=layer, blocks=torch.arange(1, BLOCKS, dtype=torch.int32, device=dev), src="gpu", dst="dram")
    torch.cuda.synchronize()
    assert st.directory().tolist() == [[0] + [1] * (BLOCKS - 1)] * L
    return st


def _rows(dev, *lead):
    g = torch.Generator(device=dev).manual_seed(len(lead))
    k = torch.randn(*lead, H, D, generator=g, device=dev).bfloat16()
    return k, -k


def _fetch(st, layer):
    """What a refetcher does: blocks that the directory has in DRAM come back."""
    st.move_blocks(layer=layer, blocks=torch.arange(BLOCKS, dtype=torch.int32, device=st.gpu_device), src="dram", dst="gpu")


@pytest.mark.parametrize("layer", [None, 1])
def test_rows_written_to_moved_blocks_stay(dev, store, layer):
    slots = torch.tensor([9, -1, 10, 20, 4 * BLOCKS, 2 ** 34 + 4, -2 ** 40], device=dev)
    k, v = _rows(dev, *((L,) if layer is None else ()), 7)
    store.write_rows(slots=slots, keys=k, values=v, layer=layer)
    written = range(L) if layer is None else [layer]
    for i in range(L):
        want = [0] + [1] * (BLOCKS - 1)
        if i in written:
            want[2] = want[5] = 0
        assert store.directory()[i].tolist() == want
    for again in (False, True):  # at once, and after a move back
        for i in written:
            ki, vi = (k[i], v[i]) if layer is None else (k, v)
            for b, r, n in ((2, 1, 0), (2, 2, 2), (5, 0, 3)):
                kb, vb = store.read_block(layer=i, block=b)
                assert kb.is_cuda and torch.equal(kb[:, r], ki[n]) and torch.equal(vb[:, r], vi[n])
            kb, vb = store.read_block(layer=i, block=2)  # rows that were there
            assert bool((kb[:, [0, 3]] == 2).all()) and bool((vb[:, [0, 3]] == 102).all())
            kb, _ = store.read_block(layer=i, block=1)
            assert bool((kb == 1).all())
            _fetch(store, i)


def test_refetcher_takes_written_blocks_as_hits(dev, store, small_config):
    from halo_amd import HALORefetcher
    k, v = _rows(dev, L, 2)
    store.write_rows(slots=torch.tensor([12, 13], device=dev), keys=k, values=v)
    r = HALORefetcher(small_config, storage=store)
    r.schedule(layer=0, predicted_indices=torch.arange(12, 20, device=dev))  # blocks 3 and 4
    r.wait()
    assert (r.hits, r.misses) == (1, 1)
    assert torch.equal(store.read_block(layer=0, block=3)[0][:, :2], k[0].transpose(0, 1))


def test_on_another_stream_and_in_a_graph(dev, store):
    k, v = _rows(dev, L, 2)
    slots = torch.tensor([28, 29], device=dev)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    store.write_rows(slots=slots, keys=k, values=v, stream=s)
    s.synchronize()
    assert store.directory()[:, 7].tolist() == [0] * L
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        store.write_rows(slots=slots, keys=k, values=v)
    for step in range(4):
        b = 1 + step
        slots.copy_(torch.tensor([4 * b, 4 * b + 3]))
        k.fill_(float(10 + step))
        g.replay()
        torch.cuda.synchronize()
        assert store.directory()[:, b].tolist() == [0] * L
        for i in range(L):
            kb, _ = store.read_block(layer=i, block=b)
            assert bool((kb[:, [0, 3]] == 10 + step).all()) and bool((kb[:, 1:3] == b).all())


def test_a_speculative_step_over_moved_blocks(dev, store):
    """Room, rows, attention and the kept path in blocks that had been moved out: the rows are read back and survive a move."""
    import halo_amd
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, owned = torch.full((1, 6), -1, dtype=torch.int32, device=dev), i32(0)
    free, n_free, lengths = i32(*reversed(range(BLOCKS))), i32(BLOCKS), i32(0)
    up = halo_amd.update_block_tables(table, owned, free, n_free, lengths + 6, lengths, block_size=BS, max_rows=6)
    assert table[0, :2].tolist() == [0, 1]
    k, v = _rows(dev, L, 6)
    q = torch.randn(6, 4, D, device=dev).bfloat16()
    for i in range(L):
        store.write_rows(slots=up.slots, keys=k[i], values=v[i], layer=i)
        out = halo_amd.tree_attention(q, *store.pool("gpu", i), table, lengths, up.cu_rows, max_nodes=6)
        assert torch.equal(out[0], v[i, 0].repeat_interleave(2, 0))
    new = halo_amd.commit_path(*store.pool(), table, lengths, i32(0, 2, 3, 5)[None], i32(4))
    assert new.tolist() == [4]
    for i in range(L):
        _fetch(store, i)
        kb, vb = store.read_block(layer=i, block=0)
        assert torch.equal(kb.transpose(0, 1), k[i, [0, 2, 3, 5]]) and torch.equal(vb.transpose(0, 1), v[i, [0, 2, 3, 5]])


def test_a_graph_does_not_make_the_directory(dev, monkeypatch):
    from halo_amd import TieredStorage
    st = TieredStorage(tiers=["gpu"], num_layers=L, num_kv_heads=H, head_dim=D, block_size=BS, dtype=torch.bfloat16,
                       device=dev, max_blocks=BLOCKS)
    k, v = _rows(dev, L, 2)
    call = lambda: st.write_rows(slots=torch.tensor([28, 29], device=dev), keys=k, values=v)  # noqa: E731
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(AssertionError, match="captured"):
            call()
    call()
    assert not st.directory().any()


def test_no_rows(dev, store):
    k, v = _rows(dev, L, 0)
    store.write_rows(slots=torch.empty(0, dtype=torch.int64, device=dev), keys=k, values=v)
    assert store.directory().tolist() == [[0] + [1] * (BLOCKS - 1)] * L


@pytest.mark.parametrize("bad", [dict(slots=torch.arange(2, dtype=torch.int32)), dict(keys=torch.zeros(L, 2, H, D)),
                                 dict(values=torch.zeros(2, H, D).bfloat16()), dict(layer=0)])
def test_refused_calls_change_nothing(dev, store, bad):
    k, v = _rows(dev, L, 2)
    args = dict(slots=torch.tensor([28, 29], device=dev), keys=k, values=v)
    with pytest.raises(AssertionError):
        store.write_rows(**{**args, **{n: t.to(dev) if torch.is_tensor(t) else t for n, t in bad.items()}})
    assert store.directory().tolist() == [[0] + [1] * (BLOCKS - 1)] * L
