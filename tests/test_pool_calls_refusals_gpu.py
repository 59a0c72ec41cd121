"""What the block-pool operators refuse on the host's tests is refused on a GPU
too, where the calls go through the host extension first, and with it off."""
from __future__ import annotations

import pytest
import torch

import test_block_pool_host as host

pytestmark = pytest.mark.gpu


def _to(dev, args):
    """The arguments with their storages on the GPU: strides and shared memory as they are."""
    moved = {}

    def move(t):
        if not torch.is_tensor(t):
            return t
        key = t.untyped_storage().data_ptr()
        if key not in moved:
            moved[key] = torch.empty(0, dtype=torch.uint8).set_(t.untyped_storage()).to(dev)
        return torch.empty(0, dtype=t.dtype, device=dev).set_(moved[key].untyped_storage(), t.storage_offset(), t.shape, t.stride())

    return {k: move(t) for k, t in args.items()}


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("name,bad", host.REFUSED, ids=lambda x: x if isinstance(x, str) else "-".join(x))
def test_refused(dev, monkeypatch, name, bad, fast):
    import halo_amd
    from halo_amd import block_pool
    assert block_pool.calls is not None
    if not fast:
        monkeypatch.setattr(block_pool, "calls", None)
    with pytest.raises(AssertionError):
        getattr(halo_amd, name)(**_to(dev, host.CALLS[name](**bad)))


@pytest.mark.parametrize("name", host.CALLS)
def test_the_plain_calls_are_taken_by_the_extension(dev, monkeypatch, name):
    import halo_amd
    from halo_amd import block_pool
    monkeypatch.setattr(block_pool.nat, "lib", lambda: pytest.fail("went through Python"))
    getattr(halo_amd, name)(**_to(dev, host.CALLS[name]()))
