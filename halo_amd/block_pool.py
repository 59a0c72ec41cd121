"""Requests over a pool of K/V blocks: block tables and slots, rows written to
their slots, drafted trees and their accepted paths.

A pool is one layer (or all layers) of a ``TieredStorage`` tier,
``(blocks, H_kv, block_size, D)`` or ``(L, blocks, H_kv, block_size, D)``.  Row
p of a request lies in row ``p % block_size`` of block
``block_table[b, p // block_size]``; ``slot = block * block_size + row``.

One speculative step of a batch, all of it on the device::

    up = update_block_tables(block_table, n_blocks, free_blocks, n_free, lengths + drafted, lengths,
                             block_size=bs, max_rows=N)            # room and slots for the drafted rows
    mask, depth = tree_layout(parents, up.cu_rows, max_nodes=n)    # row positions: lengths + depth
    for layer: append_rows(k, v, up.slots, k_pool[layer], v_pool[layer])
               tree_attention(q, k_pool[layer], v_pool[layer], block_table, lengths, up.cu_rows, mask=mask, ...)
    lengths = commit_path(k_pool, v_pool, block_table, lengths, path, n_path)   # all layers

The calls know blocks, not tiers: where a store moves blocks between tiers,
``TieredStorage.write_rows`` is ``append_rows`` with the tier directory kept.

No call waits for the device, so a step can be captured in a HIP graph; the
tensors a call changes are the caller's.  The calls run on ``stream`` (default:
the current stream of the tensors' device).

The reference stores such blocks (halo/memory_tier.py:45-60) and moves them
between tiers; it hands none to requests, so these calls have no counterpart
there.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _native as nat

MAX_NODES = 512  # nodes of one drafted tree
MAX_PATH = 64    # entries of one accepted path

_POOL = struct.Struct("<2Q4q6i")  # halo_block_pool
assert _POOL.size == 72

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


class BlockUpdate(NamedTuple):
    """What ``update_block_tables`` found: ``cu_rows`` (B + 1) int32, the new
    rows of request b are ``cu_rows[b]:cu_rows[b + 1]``; ``slots`` (max_rows)
    int64, -1 where there is none; ``ok`` (B) bool, whether b was served."""

    cu_rows: torch.Tensor
    slots: torch.Tensor
    ok: torch.Tensor


def load_calls(path=None):
    """The prebuilt host extension (halo_amd/_lib/poolcalls_build, made by
    build()) that checks, allocates and calls in C++, bound to the library; None
    when it is missing or cannot be loaded.  Its functions return None for a call
    that they do not take, which then runs (or is refused) here; an argument that
    is no tensor or number where one belongs is a TypeError there."""
    import ctypes
    import importlib.util
    import os
    if path is None:
        path = os.path.join(os.path.dirname(nat.library_path()), "poolcalls_build", "_halo_poolcalls.so")
    if not os.path.exists(path) or not nat.available():
        return None
    try:
        spec = importlib.util.spec_from_file_location("_halo_poolcalls", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.bind(*[ctypes.cast(getattr(nat.lib(), "halo_" + n), ctypes.c_void_p).value for n in
                   ("update_block_tables", "append_rows", "tree_layout", "tree_workspace_size", "tree_attn",
                    "commit_path")])
        return mod
    except (ImportError, OSError, AttributeError):
        # built against another torch, or not a loadable module: the calls are made in Python (same results, slower)
        return None


calls = load_calls()


def called(r, what: str):
    """What a function of ``calls`` returned, unless it is a status below 0."""
    if type(r) is int:
        nat.check(r, what)
    return r


class _Here:
    """Enters nothing: the call's device and stream are the current ones."""

    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_stream(device: torch.device, stream):
    """The context a call on ``device`` allocates and launches in."""
    if device.type != "cuda":
        raise AssertionError(f"the tensors must be on a GPU, not on {device}")
    if stream is not None:
        if stream.device != device:
            raise AssertionError(f"stream is on {stream.device}, the tensors on {device}")
        return torch.cuda.stream(stream)
    if device.index != torch.cuda.current_device():
        return torch.cuda.device(device)
    return _HERE


def check_ints(t: torch.Tensor, name: str, shape, device: torch.device, dtype=torch.int32) -> None:
    if t.dtype != dtype or t.device != device or tuple(t.shape) != shape or not t.is_contiguous():
        raise AssertionError(f"{name} must be a contiguous {dtype} tensor {shape} on {device}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")


def check_table(t: torch.Tensor, B: int, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.device != device or t.dim() != 2 or t.shape[0] != B or t.stride(1) != 1:
        raise AssertionError(f"block_table must be (B={B}, blocks) int32 on {device} with unit last stride, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
    if t.shape[1] < 1 or (B > 1 and t.stride(0) < t.shape[1]):
        raise AssertionError("block_table needs columns, and rows that do not overlap")


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory that two tensors span overlaps."""
    ends = []
    for t in (a, b):
        lo = t.data_ptr()
        n = t.numel() and 1 + sum((k - 1) * st for k, st in zip(t.shape, t.stride()))
        ends += [lo, lo + n * t.element_size()]
    return ends[0] < ends[3] and ends[2] < ends[1]


def pack_pool(k_pool: torch.Tensor, v_pool: torch.Tensor, *, written: bool = False) -> bytes:
    """The ``halo_block_pool`` record of K and V pools (checked); ``written``: the call changes them."""
    shape, st = k_pool.shape, k_pool.stride()
    if k_pool.dtype not in _DTYPES or v_pool.dtype != k_pool.dtype:
        raise AssertionError(f"pools must share bf16, fp16 or fp32, got {k_pool.dtype}/{v_pool.dtype}")
    if len(shape) not in (4, 5) or v_pool.shape != shape:
        raise AssertionError(f"pools must be ([L,] blocks, H_kv, block_size, D), got {tuple(shape)} and "
                             f"{tuple(v_pool.shape)}")
    if v_pool.device != k_pool.device:
        raise AssertionError("pools must be on one device")
    if v_pool.stride() != st or st[-1] != 1 or 0 in shape:
        raise AssertionError("pools must share strides, with a unit last stride, and hold rows")
    if written and (k_pool.data_ptr() == v_pool.data_ptr() or any(n > 1 and d == 0 for n, d in zip(shape, st))):
        raise AssertionError("rows that are written must have memory of their own: K and V are one pool, or expanded")
    layers, sl = (shape[0], st[0]) if len(shape) == 5 else (1, 0)
    return _POOL.pack(k_pool.data_ptr(), v_pool.data_ptr(), sl, st[-4], st[-3], st[-2], layers, shape[-4], shape[-3],
                      shape[-2], shape[-1], nat.dtype_code(k_pool.dtype))


def update_block_tables(block_table: torch.Tensor, n_blocks: torch.Tensor, free_blocks: torch.Tensor,
                        n_free: torch.Tensor, lengths: torch.Tensor, first: torch.Tensor, *, block_size: int,
                        max_rows: int, stream=None) -> BlockUpdate:
    """Gives every request the blocks its ``lengths[b]`` rows need, and the new
    rows ``first[b] .. lengths[b] - 1`` their slots.

    Changed in place: ``block_table`` (B, W) int32, of which request b owns the
    first ``n_blocks[b]`` entries; ``n_blocks`` (B); the stack
    ``free_blocks[:n_free]`` of free blocks; ``n_free`` (1), all int32.  Surplus
    blocks go back first (entries become -1; a length of 0 gives back all), then
    requests take theirs in order.  A request whose blocks do not fit the
    table's W columns, or that the free list does not cover any more, keeps what
    it has, its rows' slots are -1 and its ``ok`` is False.  New rows are
    numbered request after request; ``max_rows`` is the room for their slots
    (rows past it get none, places behind the last row are -1)."""
    if calls is not None and stream is None:
        r = calls.update_block_tables(block_table, n_blocks, free_blocks, n_free, lengths, first, block_size, max_rows)
        if r is not None:
            return BlockUpdate(*called(r, "halo_update_block_tables"))
    L = nat.lib()
    dev = block_table.device
    B = lengths.numel()
    if B < 1:
        raise AssertionError("no requests")
    check_table(block_table, B, dev)
    check_ints(n_blocks, "n_blocks", (B,), dev)
    check_ints(lengths, "lengths", (B,), dev)
    check_ints(first, "first", (B,), dev)
    check_ints(n_free, "n_free", (1,), dev)
    check_ints(free_blocks, "free_blocks", (free_blocks.numel(),), dev)
    for t, name in ((n_blocks, "n_blocks"), (n_free, "n_free"), (free_blocks, "free_blocks"), (block_table, "block_table")):
        if overlap(t, lengths) or overlap(t, first):
            raise AssertionError(f"{name} is changed: it must not share memory with lengths or first")
    if block_size < 1 or max_rows < 0:
        raise AssertionError(f"need block_size >= 1 and max_rows >= 0, got {block_size} and {max_rows}")
    with on_stream(dev, stream):
        cu_rows = torch.empty(B + 1, device=dev, dtype=torch.int32)
        slots = torch.empty(max_rows, device=dev, dtype=torch.int64)
        ok = torch.empty(B, device=dev, dtype=torch.bool)
        nat.check(L.halo_update_block_tables(
            block_table.data_ptr(), block_table.stride(0) if B > 1 else block_table.shape[1], n_blocks.data_ptr(), B,
            block_table.shape[1], free_blocks.data_ptr(), free_blocks.numel(), n_free.data_ptr(), lengths.data_ptr(),
            first.data_ptr(), block_size, max_rows, cu_rows.data_ptr(), slots.data_ptr(), ok.data_ptr(),
            nat.stream_ptr()), "halo_update_block_tables")
    return BlockUpdate(cu_rows, slots, ok)


def append_rows(k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor, k_pool: torch.Tensor,
                v_pool: torch.Tensor, *, stream=None) -> None:
    """Writes row i of ``k_new``/``v_new`` ([L,] N, H_kv, D) to slot
    ``slots[i]`` (int64) of the pools ([L,] blocks, H_kv, block_size, D), in
    every layer.  Rows whose slot is negative or past the pool are skipped.
    Slots must differ: which of two rows with one slot stays is not defined."""
    if calls is not None and stream is None:
        r = calls.append_rows(k_new, v_new, slots, k_pool, v_pool)
        if r is not None:
            called(r, "halo_append_rows")
            return
    L = nat.lib()
    pool = pack_pool(k_pool, v_pool, written=True)
    dev = k_pool.device
    five = k_pool.dim() == 5
    want = k_pool.shape[:1] * five + slots.shape + (k_pool.shape[-3], k_pool.shape[-1])
    for t, name in ((k_new, "k_new"), (v_new, "v_new")):
        if t.dtype != k_pool.dtype or t.device != dev or t.shape != want or t.stride(-1) != 1:
            raise AssertionError(f"{name} must be {tuple(want)} {k_pool.dtype} on {dev} with unit last stride, got "
                                 f"{tuple(t.shape)} {t.dtype} on {t.device}")
        if overlap(t, k_pool) or overlap(t, v_pool):
            raise AssertionError(f"{name} must not share memory with the pools")
    check_ints(slots, "slots", (slots.numel(),), dev, torch.int64)
    ks, vs = k_new.stride(), v_new.stride()
    with on_stream(dev, stream):
        nat.check(L.halo_append_rows(pool, k_new.data_ptr(), ks[0] if five else 0, ks[-3], ks[-2], v_new.data_ptr(),
                                     vs[0] if five else 0, vs[-3], vs[-2], slots.data_ptr(), slots.numel(),
                                     nat.stream_ptr()), "halo_append_rows")


def tree_layout(parents: torch.Tensor, cu_nodes: torch.Tensor, *, max_nodes: int,
                mask: Optional[torch.Tensor] = None, depth: Optional[torch.Tensor] = None, stream=None):
    """Ancestor masks and depths of drafted trees.

    ``parents`` (N) int32: node i of request b is entry ``cu_nodes[b] + i``
    (``cu_nodes`` (B + 1) int32) and holds its parent's number in the same tree;
    a value that names no earlier node makes it a root.  ``max_nodes`` (<= 512)
    is the largest tree.  Returns ``mask`` (N, ceil(max_nodes / 64)) int64, bit
    j of a node's words set for itself and its ancestors, and ``depth`` (N)
    int32, the number of ancestors.  Entries of no tree (a padded batch) are not
    written; ``mask`` and ``depth`` may be given."""
    if calls is not None and stream is None and mask is None and depth is None:
        r = calls.tree_layout(parents, cu_nodes, max_nodes)
        if r is not None:
            return called(r, "halo_tree_layout")
    L = nat.lib()
    dev = parents.device
    N, B, words = parents.numel(), cu_nodes.numel() - 1, (max_nodes + 63) // 64
    if not 1 <= max_nodes <= MAX_NODES:
        raise AssertionError(f"max_nodes must be in [1, {MAX_NODES}], got {max_nodes}")
    if B < 1:
        raise AssertionError("cu_nodes needs an entry more than there are requests")
    check_ints(parents, "parents", (N,), dev)
    check_ints(cu_nodes, "cu_nodes", (B + 1,), dev)
    if mask is not None:
        check_ints(mask, "mask", (N, words), dev, torch.int64)
    if depth is not None:
        check_ints(depth, "depth", (N,), dev)
    with on_stream(dev, stream):
        if mask is None:
            mask = torch.empty((N, words), device=dev, dtype=torch.int64)
        if depth is None:
            depth = torch.empty(N, device=dev, dtype=torch.int32)
        if N:
            nat.check(L.halo_tree_layout(parents.data_ptr(), cu_nodes.data_ptr(), B, N, max_nodes, mask.data_ptr(),
                                         words, depth.data_ptr(), nat.stream_ptr()), "halo_tree_layout")
    return mask, depth


def commit_path(k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                path: torch.Tensor, n_path: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """Keeps the accepted path of each request's drafted tree: row
    ``lengths[b] + j`` of every layer of the pools receives what row
    ``lengths[b] + path[b, j]`` held, for ``j < n_path[b]``.

    ``path`` (B, P <= 64) int32 rises; it ends at the first entry that does not,
    or whose row the table does not hold.  Rows behind the committed ones lie in
    blocks that no other request has (committed blocks may be shared).  Returns the new lengths (B) int32,
    in ``out`` if given (memory of its own, not ``lengths``)."""
    if calls is not None and stream is None:
        r = calls.commit_path(k_pool, v_pool, block_table, lengths, path, n_path, out)
        if r is not None:
            return called(r, "halo_commit_path")
    L = nat.lib()
    pool = pack_pool(k_pool, v_pool, written=True)
    dev = k_pool.device
    B = lengths.numel()
    if B < 1 or path.dim() != 2 or not 1 <= path.shape[1] <= MAX_PATH:
        raise AssertionError(f"path must be (B, P) with 1 <= P <= {MAX_PATH}, got {tuple(path.shape)}")
    check_table(block_table, B, dev)
    check_ints(lengths, "lengths", (B,), dev)
    check_ints(path, "path", (B, path.shape[1]), dev)
    check_ints(n_path, "n_path", (B,), dev)
    if out is not None:
        check_ints(out, "out", (B,), dev)
        if any(overlap(out, t) for t in (lengths, path, n_path, block_table)):
            raise AssertionError("out must not share memory with what is read")
    with on_stream(dev, stream):
        if out is None:
            out = torch.empty(B, device=dev, dtype=torch.int32)
        nat.check(L.halo_commit_path(pool, block_table.data_ptr(),
                                     block_table.stride(0) if B > 1 else block_table.shape[1], B, block_table.shape[1],
                                     lengths.data_ptr(), path.data_ptr(), path.shape[1], path.shape[1],
                                     n_path.data_ptr(), out.data_ptr(), nat.stream_ptr()), "halo_commit_path")
    return out
