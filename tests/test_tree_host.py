"""Refusals of tree attention's outputs, without a GPU."""
from __future__ import annotations

import pytest
import torch

from test_block_pool_host import _attend, lib  # noqa: F401


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.int64, torch.int16, torch.uint8, torch.bool, torch.complex64])
def test_outputs_of_other_types_are_refused(lib, dtype):  # noqa: F811
    """Not bf16, fp16 or fp32: rows of no request would come back changed, and others cut to whole numbers."""
    import halo_amd
    for kw in (dict(out=torch.zeros(5, 4, 64, dtype=dtype)), dict(out_dtype=dtype),
               dict(out=torch.zeros(5, 4, 64, dtype=dtype), out_dtype=dtype)):
        with pytest.raises(AssertionError, match="out"):
            halo_amd.tree_attention(**_attend(**kw))
    assert lib.calls == []


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_outputs_of_the_three_types_are_taken(lib, dtype):  # noqa: F811
    import halo_amd
    assert halo_amd.tree_attention(**_attend(out_dtype=dtype)).dtype == dtype
    out = torch.zeros(5, 4, 64, dtype=dtype)
    assert halo_amd.tree_attention(**_attend(out=out)) is out
    assert len(lib.calls) == 2
