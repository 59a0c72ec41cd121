"""Attention of drafted token trees, and of prompts, over a paged cache.

``tree_attention`` verifies the drafted tokens of a batch in one call: every
node attends its request's committed rows and, of the tree's own rows behind
them, itself and its ancestors.  K and V lie in the blocks of a pool
(``halo_amd.block_pool``), so the requests' lengths and trees may differ freely
and change from call to call without a host plan: the lengths are read on the
device, and a captured call follows them.  With one node a request it is a
paged decode step; without masks, a causal block of new rows.
``chunk_attention`` is the causal form for prompts, with any number of rows.

The reference attends a chunk list with one row or one causal block a call
(halo/kv_cache_chunked.py:571-964); it has no drafted trees.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native as nat
from . import block_pool as pool_calls
from .block_pool import _DTYPES, MAX_NODES, check_ints, check_table, on_stream, overlap, pack_pool

PLAN_REQUESTS = 4096  # requests that the plan of a call of chunks holds


def tree_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                   lengths: torch.Tensor, cu_nodes: torch.Tensor, *, max_nodes: int,
                   mask: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                   out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   lse: Optional[torch.Tensor] = None, return_lse: bool = False, stream=None):
    """q (N, H, D) bf16, fp16 or fp32, D 64 or 128; pools (blocks, H_kv,
    block_size, D) of the same dtype; ``block_table`` (B, W), ``lengths`` (B)
    and ``cu_nodes`` (B + 1) int32.

    Node i of request b is row ``cu_nodes[b] + i``; it attends the rows
    ``[0, lengths[b])`` and of the rows ``lengths[b] + j`` those whose bit j is
    set in its row of ``mask`` (N, >= ceil(max_nodes / 64)) int64, the form
    ``tree_layout`` gives; without a mask, ``j <= i``.  ``max_nodes`` (<= 512) is
    the largest tree; further nodes of a request are left out.  Rows in blocks
    outside the pool (a table entry of -1, say) are not attended, a node that
    attends nothing has out 0 and lse -inf, and what a node does not attend has
    no part in its output, NaN and infinities included.

    Returns out (N, H, D) in ``out_dtype`` (bf16, fp16 or fp32; default
    q.dtype), and with ``return_lse`` lse (N, H) fp32, both in ``out`` and ``lse``
    if given; rows of no request keep what they hold there.  The softmax and all
    sums are fp32; for 16-bit pools its weights are rounded once to the pool's
    type (fp16 weights below 2^-21 of the largest are off by at most 2^-32 of it, where
    scores reach 2^24 2^-29; beyond 2^24 fp16 results are finite up to 2^29, but
    their accuracy is not covered).  Equal calls give equal bits; where
    a request's rows are cut, and so its last bits, goes by all the requests of
    the call.  No gradient is kept."""
    if pool_calls.calls is not None and stream is None and out_dtype is None:
        r = pool_calls.calls.tree_attention(q, k_pool, v_pool, block_table, lengths, cu_nodes, max_nodes, mask, scale,
                                            out, lse, return_lse)
        if r is not None:
            return pool_calls.called(r, "halo_tree_attn")
    nat.lib()
    if not 1 <= max_nodes <= MAX_NODES:
        raise AssertionError(f"max_nodes must be in [1, {MAX_NODES}], got {max_nodes}")
    return _attend(q, k_pool, v_pool, block_table, lengths, cu_nodes, "cu_nodes", max_nodes, mask, False, scale, out,
                   out_dtype, lse, return_lse, stream)


def chunk_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor,
                    lengths: torch.Tensor, cu_rows: torch.Tensor, *, max_rows: int, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                    lse: Optional[torch.Tensor] = None, return_lse: bool = False, stream=None):
    """Attention of prompts, or slices of them, over the blocks they have been
    written to: q (N, H, D), pools, ``block_table``, ``lengths`` and the results
    as in ``tree_attention``.

    Row i of request b is row ``cu_rows[b] + i`` (``cu_rows`` (B + 1) int32) and
    attends the rows ``[0, lengths[b] + i]``: what the request held before, the
    new rows before it and itself, all of them in the pool already
    (``append_rows``, ``rotate_rows``).  Requests may have any numbers of new
    rows, none and one among them; ``max_rows`` is the largest (further rows are
    left out).  The lengths are read on the device, so a captured call follows
    them.  Calls of more than 4096 requests have at most 512 rows each; N times
    H / H_kv stays below 2^30."""
    if pool_calls.calls is not None and stream is None and out_dtype is None:
        r = pool_calls.calls.chunk_attention(q, k_pool, v_pool, block_table, lengths, cu_rows, max_rows, scale, out, lse,
                                             return_lse)
        if r is not None:
            return pool_calls.called(r, "halo_chunk_attn")
    nat.lib()
    if max_rows < 1:
        raise AssertionError(f"max_rows must be at least 1, got {max_rows}")
    if q.dim():  # no request has more rows than there are
        max_rows = min(max_rows, max(q.shape[0], 1))
    # the plan of chunks holds PLAN_REQUESTS; rows of more are nodes of trees without masks
    chunk = lengths.numel() <= PLAN_REQUESTS or max_rows > MAX_NODES
    return _attend(q, k_pool, v_pool, block_table, lengths, cu_rows, "cu_rows", max_rows, None, chunk, scale, out, out_dtype, lse,
                   return_lse, stream)


def _attend(q, k_pool, v_pool, block_table, lengths, cu, cu_name, max_nodes, mask, chunk, scale, out, out_dtype, lse,
            return_lse, stream):
    L = nat.lib()
    if q.dim() != 3:
        raise AssertionError(f"q must be (N, H, D), got {tuple(q.shape)}")
    N, H, D = q.shape
    dev = q.device
    pool = pack_pool(k_pool, v_pool)
    shape = k_pool.shape
    if len(shape) != 4 or shape[-1] != D or k_pool.dtype != q.dtype or k_pool.device != dev:
        raise AssertionError(f"pools must be (blocks, H_kv, block_size, {D}) {q.dtype} on {dev}, got {tuple(shape)} "
                             f"{k_pool.dtype} on {k_pool.device}")
    if D not in (64, 128):
        raise AssertionError(f"head_dim must be 64 or 128, got {D}")
    if H == 0 or H % shape[1]:
        raise AssertionError(f"head count mismatch: q has {H}, kv has {shape[1]}")
    B = lengths.numel()
    if B < 1:
        raise AssertionError("no requests")
    check_table(block_table, B, dev)
    check_ints(lengths, "lengths", (B,), dev)
    check_ints(cu, cu_name, (B + 1,), dev)
    words = 0
    if mask is not None:
        if mask.dtype != torch.int64 or mask.device != dev or mask.dim() != 2 or mask.shape[0] != N \
                or mask.shape[1] * 64 < max_nodes or not mask.is_contiguous():
            raise AssertionError(f"mask must be contiguous ({N}, >= {(max_nodes + 63) // 64}) int64 on {dev}, got "
                                 f"{mask.dtype} {tuple(mask.shape)} on {mask.device}")
        words = mask.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise AssertionError(f"scale must be positive and finite, got {scale}")
    if out_dtype is not None and out_dtype not in _DTYPES:
        raise AssertionError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
    if out is not None and out.dtype not in _DTYPES:
        # its copy in fp32 could not hold the rows that are not written
        raise AssertionError(f"out must be bf16, fp16 or fp32, got {out.dtype}")
    if out is not None and (out.shape != q.shape or out.device != dev or out.stride(-1) != 1
                            or out.dtype != (out_dtype or out.dtype)
                            or any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride()))):
        raise AssertionError(f"out must be {tuple(q.shape)} on {dev} with unit last stride, not expanded")
    if out is not None and (overlap(out, q) or overlap(out, k_pool) or overlap(out, v_pool)):
        raise AssertionError("out must not share memory with q or the pools")
    if lse is not None and (lse.shape != (N, H) or lse.dtype != torch.float32 or lse.device != dev
                            or not lse.is_contiguous()):
        raise AssertionError(f"lse must be contiguous float32 {(N, H)} on {dev}")
    if lse is not None and any(overlap(lse, t) for t in (q, k_pool, v_pool, out) if t is not None):
        raise AssertionError("lse must not share memory with q, the pools or out")
    with on_stream(dev, stream):
        qs = q.stride()
        per = 16 // q.element_size()
        if qs[2] != 1 or qs[0] % per or qs[1] % per or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            qs = q.stride()
        want = out.dtype if out is not None else out_dtype or q.dtype
        # the kernel writes q's type or fp32, rows aligned to four elements
        o = out
        if out is None or (want != q.dtype and want != torch.float32) or out.data_ptr() % (4 * out.element_size()) \
                or out.stride(0) % 4 or out.stride(1) % 4:
            o = torch.empty((N, H, D), device=dev, dtype=want if want == q.dtype else torch.float32)
            if out is not None:
                o.copy_(out)  # for the rows that are not written
        if return_lse and lse is None:
            lse = torch.empty((N, H), device=dev, dtype=torch.float32)
        W = block_table.shape[1]
        dt = nat.dtype_code(q.dtype)
        if chunk:
            nbytes = L.halo_chunk_workspace_size(dt, B, N, H, shape[1], D, W * shape[2], max_nodes)
        else:
            nbytes = L.halo_tree_workspace_size(dt, B, H, shape[1], D, W * shape[2], max_nodes)
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
        os_ = o.stride()
        head = (pool, q.data_ptr(), qs[0], qs[1], N, H, block_table.data_ptr(), block_table.stride(0) if B > 1 else W, B, W,
                lengths.data_ptr(), cu.data_ptr(), max_nodes)
        tail = (scale, o.data_ptr(), os_[0], os_[1], nat.dtype_code(o.dtype), nat.ptr(lse), nat.ptr(ws), nbytes,
                nat.stream_ptr())
        if chunk:
            nat.check(L.halo_chunk_attn(*head, *tail), "halo_chunk_attn")
        else:
            nat.check(L.halo_tree_attn(*head, nat.ptr(mask), words, *tail), "halo_tree_attn")
        if out is None:
            out = o if o.dtype == want else o.to(want)
        elif o is not out:
            out.copy_(o)
    return (out, lse) if return_lse else out
