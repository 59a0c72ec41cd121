"""The operators around the block pool through the host extension and through
Python: same results, on the current stream, and refusals as they are."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _calls(dev, seed=0):
    """A call of each in a few forms; everything they return and change."""
    import halo_amd
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    H, Hk, D, bs, P, N = 8, 2, 64, 16, 120, 700
    kp, vp = rand(2, P, Hk, bs, D), rand(2, P, Hk, bs, D)
    table = torch.full((3, 60), -1, dtype=I32, device=dev)
    owned, n_free = i32([0, 0, 0]), i32([P])
    free = torch.randperm(P, generator=g, device=dev).to(I32)
    shared = torch.zeros(P, dtype=I32, device=dev)
    lengths = i32([5, 300, 0])
    new = i32([600, 100, 0])
    up = halo_amd.update_block_tables(table, owned, free, n_free, lengths + new, lengths, block_size=bs, max_rows=N)
    angle = torch.rand(1000, D // 2, generator=g, device=dev) * 6
    qkv = rand(N, H + 2 * Hk, D)
    w = rand(D)
    pos = torch.arange(N, device=dev)
    args = (qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:], pos, angle.cos(), angle.sin(), up.slots, kp[0], vp[0])
    q = halo_amd.rotate_rows(*args, q_norm=w, k_norm=w.float())
    q2 = halo_amd.rotate_rows(*args[:7], kp[1], vp[1], interleaved=True, eps=1e-5)
    out, lse = halo_amd.chunk_attention(q, kp[0], vp[0], table, lengths, up.cu_rows, max_rows=600, return_lse=True)
    mine = halo_amd.chunk_attention(q2, kp[1], vp[1], table, lengths, up.cu_rows, max_rows=600, out=torch.empty_like(q), scale=0.3)
    few = halo_amd.chunk_attention(q[:40], kp[0], vp[0], table, lengths, i32([0, 17, 40, 40]), max_rows=23)
    lens, ok = halo_amd.fork_blocks(table, owned, free, n_free, shared, lengths + new, i32([0, 1, 1]), kp, vp)
    lens2, ok2 = halo_amd.fork_blocks(table, owned, free, n_free, shared, lens, i32([-1, 2, 2]), kp, vp)
    new_id, used = halo_amd.compact_blocks(table, owned, free, n_free, shared, kp, vp)
    probs = torch.softmax(torch.randn(9, 500, generator=g, device=dev) * 2, 1)
    draft = torch.softmax(torch.randn(9, 500, generator=g, device=dev) * 2, 1)
    tree = dict(tokens=torch.randint(0, 500, (9,), generator=g, device=dev), parents=i32([-1, 0, 0, 1, 0, -1, 0, 1, 2]),
                cu_nodes=i32([0, 5, 9]), probs=probs, accept=torch.rand(9, generator=g, device=dev),
                sample=torch.rand(2, generator=g, device=dev), max_nodes=5)
    v = [x for kw in ({}, dict(draft_probs=draft), dict(draft_probs=draft, replacement=False, max_path=2))
         for x in halo_amd.verify_tree(**tree, **kw)]
    return [q, q2, out[:N], lse, mine, few, lens, ok, lens2, ok2, new_id, used, table, owned, free, n_free, shared, kp, vp, *v]


def test_extension_and_python_agree(dev, monkeypatch):
    from halo_amd import block_pool
    assert block_pool.calls is not None, "halo_amd/_lib/poolcalls_build is not built"
    fast = _calls(dev)
    monkeypatch.setattr(block_pool, "calls", None)
    slow = _calls(dev)
    assert len(fast) == len(slow)
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_calls_run_on_the_current_stream(dev):
    want = _calls(dev)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _calls(dev)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_extension_leaves_refusals_to_python(dev):
    import halo_amd
    i32 = lambda *x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    kp, vp = torch.zeros(4, 2, 16, 64, device=dev), torch.zeros(4, 2, 16, 64, device=dev)
    table, one, free, shared = i32(0, 1, 2)[None], i32(1), i32(3, 0, 0), torch.zeros(4, dtype=I32, device=dev)
    q, kv = torch.zeros(1, 4, 64, device=dev), torch.zeros(1, 2, 64, device=dev)
    trig, slot = torch.ones(3, 32, device=dev), torch.zeros(1, dtype=torch.int64, device=dev)
    with pytest.raises(AssertionError):
        halo_amd.fork_blocks(table, one, free, i32(1), shared, one, i32(0), kp, vp)  # lengths is n_blocks
    with pytest.raises(AssertionError):
        halo_amd.fork_blocks(table, one, free, i32(1), shared[:3], i32(5), i32(0), kp, vp)
    with pytest.raises(AssertionError):
        halo_amd.compact_blocks(table, one, free, i32(1), shared, kp, kp)
    with pytest.raises(AssertionError):
        halo_amd.rotate_rows(q, kv, kv, slot, trig[:, :20].contiguous(), trig[:, :20].contiguous(), slot, kp, vp)
    with pytest.raises(AssertionError):
        halo_amd.rotate_rows(q.half(), kv, kv, slot, trig, trig, slot, kp, vp)
    with pytest.raises(AssertionError):
        halo_amd.chunk_attention(q, kp, vp, table, one, i32(0, 1), max_rows=0)
    with pytest.raises(AssertionError):
        halo_amd.verify_tree(slot, one, i32(0, 1), trig[:1], trig[0, :1], trig[0, :2], max_nodes=1)
    with pytest.raises(AssertionError):
        halo_amd.verify_tree(slot.cpu(), one, i32(0, 1), trig[:1], trig[0, :1], trig[0, :1], max_nodes=1)


def test_calls_without_rows_or_nodes(dev):
    import halo_amd
    i32 = lambda *x: torch.tensor(x, dtype=I32, device=dev)  # noqa: E731
    kp, vp = torch.zeros(4, 2, 16, 64, device=dev), torch.zeros(4, 2, 16, 64, device=dev)
    out, lse = halo_amd.chunk_attention(torch.zeros(0, 4, 64, device=dev), kp, vp, i32(0, 1)[None], i32(7), i32(0, 0), max_rows=9,
                                        return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    e = torch.zeros(0, device=dev)
    v = halo_amd.verify_tree(e.long(), e.int(), i32(0, 0, 0), torch.zeros(0, 11, device=dev), e, torch.zeros(2, device=dev), max_nodes=3)
    assert v.path.tolist() == [[-1] * 3] * 2 and v.n_path.tolist() == [0, 0] and v.token.tolist() == [-1, -1]
