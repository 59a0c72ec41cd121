"""Tree attention's forms of output, and requests in other company, on the GPU.
Tolerances as in test_tree_pipeline_gpu.py."""
from __future__ import annotations

import pytest
import torch

import tree_launch
from test_tree_pipeline_gpu import BF16, F16, F32, check

pytestmark = pytest.mark.gpu


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


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_request_alone_and_among_others(dev, dtype):
    """Each is right by itself; their last bits may differ, since the cuts go by all the requests of a call."""
    b = tree_launch.Batch(dev, lengths=[3000, 17, 1200, 0, 5000], nodes=[5, 9, 2, 12, 7], H=8, Hk=2, D=128, bs=16, dtype=dtype, seed=4)
    out, lse = b.run()
    for i in (0, 1, 3, 4):
        lo, hi = sum(b.nodes[:i]), sum(b.nodes[:i + 1])
        one = tree_launch.Batch.__new__(tree_launch.Batch)
        one.__dict__.update(b.__dict__, lengths=[b.lengths[i]], nodes=[b.nodes[i]], max_nodes=b.nodes[i])
        a = b.args
        one.args = dict(a, q=a["q"][lo:hi], mask=a["mask"][lo:hi], block_table=a["block_table"][i:i + 1], lengths=a["lengths"][i:i + 1],
                        cu_nodes=a["cu_nodes"].new_tensor([0, hi - lo]))
        exact = one.exact()
        check(one, *one.run(), exact)
        check(one, out, lse, exact, rows=slice(lo, hi))
