"""The block-pool operators' calls through the host extension and through
Python: same results, on the current stream, and refusals as they are."""
from __future__ import annotations

import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _step(dev, seed=0):
    """One step's calls; everything they return and change."""
    import halo_amd
    g = torch.Generator(device=dev).manual_seed(seed)
    B, H, Hk, D, bs, L = 3, 8, 2, 64, 16, 2
    table = torch.full((B, 40), -1, dtype=I32, device=dev)
    owned, n_free = torch.zeros(B, dtype=I32, device=dev), torch.full((1,), 100, dtype=I32, device=dev)
    free = torch.randperm(100, generator=g, device=dev).to(I32)
    lengths = torch.tensor([5, 300, 0], dtype=I32, device=dev)
    new = torch.tensor([9, 3, 20], dtype=I32, device=dev)
    up = halo_amd.update_block_tables(table, owned, free, n_free, lengths + new, lengths, block_size=bs, max_rows=40)
    parents = torch.randint(-1, 3, (32,), generator=g, device=dev).to(I32)
    mask, depth = halo_amd.tree_layout(parents, up.cu_rows, max_nodes=20)
    k, v, kp, vp = (torch.randn(s, generator=g, device=dev).to(torch.bfloat16) for s in
                    2 * [(L, 40, Hk, D)] + 2 * [(L, 100, Hk, bs, D)])
    halo_amd.append_rows(k, v, up.slots, kp, vp)
    q = torch.randn((32, H, D), generator=g, device=dev).to(torch.bfloat16)
    out, lse = halo_amd.tree_attention(q, kp[1], vp[1], table, lengths, up.cu_rows, mask=mask, max_nodes=20,
                                       return_lse=True)
    mine = halo_amd.tree_attention(q, kp[0], vp[0], table, lengths, up.cu_rows, max_nodes=20,
                                   out=torch.empty_like(q), scale=0.3)
    path = torch.tensor([[0, 2, 5], [1, 2, 0], [3, 8, 19]], dtype=I32, device=dev)
    kept = halo_amd.commit_path(kp, vp, table, lengths, path, torch.tensor([3, 3, 2], dtype=I32, device=dev))
    again = halo_amd.commit_path(kp, vp, table, lengths, path, torch.tensor([1, 0, 0], dtype=I32, device=dev),
                                 out=torch.empty_like(lengths))
    return [table, owned, free, n_free, *up, mask, depth, kp, vp, out, lse, mine, kept, again]


def test_extension_and_python_agree(dev, monkeypatch):
    from halo_amd import block_pool
    assert block_pool.calls is not None, "halo_amd/_lib/poolcalls_build is not built"
    fast = _step(dev)
    monkeypatch.setattr(block_pool, "calls", None)
    slow = _step(dev)
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_calls_run_on_the_current_stream(dev):
    from halo_amd import block_pool
    assert block_pool.calls is not None
    want = _step(dev)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _step(dev)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_extension_leaves_refusals_to_python(dev):
    import halo_amd
    q = torch.zeros(4, 4, 64, device=dev)
    kp, vp = torch.zeros(3, 2, 16, 64, device=dev), torch.zeros(3, 2, 16, 64, device=dev)
    t, one, cu = (torch.zeros(1, 3, dtype=I32, device=dev), torch.ones(1, dtype=I32, device=dev),
                  torch.tensor([0, 4], dtype=I32, device=dev))
    ok = dict(q=q, k_pool=kp, v_pool=vp, block_table=t, lengths=one, cu_nodes=cu, max_nodes=4)
    halo_amd.tree_attention(**ok)
    for bad in (dict(q=q[:, :3]), dict(q=q.half()), dict(k_pool=kp.cpu()), dict(max_nodes=0), dict(scale=math.inf),
                dict(lengths=one.long()), dict(cu_nodes=cu[:1]), dict(out=q), dict(mask=cu)):
        with pytest.raises(AssertionError):
            halo_amd.tree_attention(**{**ok, **bad})
    with pytest.raises(AssertionError):
        halo_amd.append_rows(kp[0].transpose(0, 1), vp[0].transpose(0, 1), torch.arange(16, device=dev), kp, vp)
    with pytest.raises(AssertionError):
        halo_amd.append_rows(q[:, :2], q[:, :2], torch.arange(4, device=dev), kp, kp)
    with pytest.raises(AssertionError):
        halo_amd.commit_path(kp, vp, t, one, torch.zeros(1, 65, dtype=I32, device=dev), one)
    with pytest.raises(AssertionError):
        halo_amd.commit_path(kp, vp, t, one, cu[None], one, out=one)
    with pytest.raises(AssertionError):
        halo_amd.update_block_tables(t, one, torch.arange(3, dtype=I32, device=dev), one, one, one, block_size=16,
                                     max_rows=1)


def test_missing_or_broken_extension_is_not_fatal(dev, tmp_path):
    from halo_amd.block_pool import load_calls
    assert load_calls(os.fspath(tmp_path / "no.so")) is None
    bad = tmp_path / "_halo_poolcalls.so"
    bad.write_bytes(b"not a library")
    assert load_calls(os.fspath(bad)) is None
