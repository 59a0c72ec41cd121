"""``TieredStorage.write_rows`` without a GPU: what it refuses."""
from __future__ import annotations

import pytest
import torch


def test_a_store_on_the_host_is_refused(storage_factory, monkeypatch):
    from halo_amd import block_pool
    monkeypatch.setattr(block_pool.nat, "lib", lambda: None)
    st = storage_factory(head_dim=64)
    k, v = st.pool()
    k.zero_(), v.zero_()
    st.directory().fill_(1)
    with pytest.raises(AssertionError, match="GPU"):
        st.write_rows(slots=torch.arange(3), keys=torch.ones(2, 3, 2, 64), values=torch.ones(2, 3, 2, 64))
    assert not k.any() and not v.any() and bool((st.directory() == 1).all())


def test_without_a_gpu_tier_there_is_no_pool():
    from halo_amd import TieredStorage
    st = TieredStorage(tiers=["dram"], num_layers=1, num_kv_heads=1, head_dim=64, block_size=4, dtype=torch.float32,
                       device="cpu", max_blocks=2)
    with pytest.raises(ValueError):
        st.write_rows(slots=torch.arange(3), keys=torch.ones(3, 1, 64), values=torch.ones(3, 1, 64), layer=0)
