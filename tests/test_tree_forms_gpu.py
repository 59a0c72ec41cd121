"""Tree attention's forms of output on the GPU."""
from __future__ import annotations

import pytest
import torch

import tree_launch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("form", ["plain", "odd start", "odd rows"])
def test_rows_of_no_request_keep_what_they_hold(dev, dtype, out_dtype, form):
    """A padded batch: outputs of each type and alignment, through a copy where the kernels cannot write them."""
    import halo_amd
    b = tree_launch.Batch(dev, lengths=[300, 20], nodes=[5, 3], H=8, Hk=2, D=64, bs=16, dtype=dtype, seed=6)
    want = b.run()
    q = torch.cat([b.args["q"], b.args["q"][:4]])
    mask = torch.cat([b.args["mask"], b.args["mask"][:4]])
    shape, cut = {"plain": ((12, 8, 64), slice(None)), "odd start": ((12, 8, 66), slice(1, 65)), "odd rows": ((12, 8, 65), slice(0, 64))}[form]
    held = (torch.arange(12 * 8 * shape[2], device=dev, dtype=torch.float32).view(shape) % 251 - 125).to(out_dtype)
    held[9, 3, 5:9] = torch.tensor([float("inf"), float("-inf"), 0.0, -0.0], device=dev, dtype=out_dtype)
    out = held.clone()[..., cut]
    lse = torch.full((12, 8), 7.0, device=dev)
    got = halo_amd.tree_attention(**{**b.args, "q": q, "mask": mask}, max_nodes=b.max_nodes, out=out, lse=lse, return_lse=True)
    assert got[0] is out and got[1] is lse
    assert torch.equal(out[8:], held[8:, :, cut]) and bool((lse[8:] == 7).all())
    assert torch.equal(lse[:8], want[1])
    full = b.run(out_dtype=torch.float32)[0]
    assert torch.equal(out[:8], full.to(out_dtype)) and torch.equal(full.to(dtype), want[0])
