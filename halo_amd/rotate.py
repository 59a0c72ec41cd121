"""Rows on their way into a paged cache: heads of queries and keys normed and
rotated, keys and values written to their slots, in one pass over the rows.

What a model does between its projections and ``chunk_attention`` or
``tree_attention``.  The reference leaves the norm and the rotation to the model
and attends what it is handed (halo/policy.py:321-478); writing the rows is
``append_rows``.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _native as nat
from . import block_pool as pool_calls
from .block_pool import check_ints, on_stream, overlap, pack_pool


def rotate_rows(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor,
                sin: torch.Tensor, slots: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, *,
                q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                interleaved: bool = False, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """q (N, H, D), k and v (N, H_kv, D) of the pools' dtype (bf16, fp16 or
    fp32; D 64 or 128), any row and head strides; ``positions`` (N) int64 or int32;
    ``cos`` and ``sin`` (positions, R / 2) fp32, R a multiple of 16 up to D;
    ``slots`` (N) int64; pools (blocks, H_kv, block_size, D).

    Each head of q and k is normed where its weight (D, of the rows' dtype or
    fp32) is given, ``y = x w / sqrt(mean(x^2) + eps)``, and its first R channels
    are rotated by the row's position: the pairs (j, j + R/2), or (2j, 2j + 1) if
    ``interleaved``, become ``(a cos - b sin, b cos + a sin)``.  k and v go to slot
    ``slots[i]`` of the pools; rows whose slot is negative or past the pool are
    not kept.  Returns q, in ``out`` if given (which may be q itself, whose heads
    then are no part of k or v).  All of it
    is fp32, rounded once at the end.  A position outside the table makes the
    rotated channels NaN.  Slots must differ, as in ``append_rows``.  No gradient
    is kept."""
    if pool_calls.calls is not None and stream is None and out is None:
        r = pool_calls.calls.rotate_rows(q, k, v, positions, cos, sin, slots, k_pool, v_pool, q_norm, k_norm, eps, interleaved)
        if r is not None:
            return pool_calls.called(r, "halo_rotate_rows")
    L = nat.lib()
    pool = pack_pool(k_pool, v_pool, written=True)
    dev, dtype = k_pool.device, k_pool.dtype
    if k_pool.dim() != 4:
        raise AssertionError(f"pools must be (blocks, H_kv, block_size, D), got {tuple(k_pool.shape)}")
    H_kv, D = k_pool.shape[1], k_pool.shape[3]
    if D not in (64, 128):
        raise AssertionError(f"head_dim must be 64 or 128, got {D}")
    N = slots.numel()
    if q.dim() != 3 or q.shape[0] != N or q.shape[1] < 1 or q.shape[2] != D or q.dtype != dtype or q.device != dev:
        raise AssertionError(f"q must be ({N}, H, {D}) {dtype} on {dev}, got {tuple(q.shape)} {q.dtype} on {q.device}")
    for t, name in ((k, "k"), (v, "v")):
        if t.shape != (N, H_kv, D) or t.dtype != dtype or t.device != dev:
            raise AssertionError(f"{name} must be {(N, H_kv, D)} {dtype} on {dev}, got {tuple(t.shape)} {t.dtype} on "
                                 f"{t.device}")
        if overlap(t, k_pool) or overlap(t, v_pool):
            raise AssertionError(f"{name} must not share memory with the pools")
    if overlap(q, k_pool) or overlap(q, v_pool):
        raise AssertionError("q must not share memory with the pools")
    check_ints(slots, "slots", (N,), dev, torch.int64)
    check_ints(positions, "positions", (N,), dev, torch.int32 if positions.dtype == torch.int32 else torch.int64)
    for t, name in ((cos, "cos"), (sin, "sin")):
        if t.dtype != torch.float32 or t.device != dev or t.dim() != 2 or t.shape != cos.shape or not t.is_contiguous():
            raise AssertionError(f"{name} must be contiguous float32 (positions, R / 2) on {dev}, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
    R = 2 * cos.shape[1]
    if cos.shape[0] < 1 or not 16 <= R <= D or R % 16:
        raise AssertionError(f"the rotated channels must be a multiple of 16 up to {D}, got {R} of {cos.shape[0]} positions")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None and (t.shape != (D,) or t.dtype not in (dtype, torch.float32) or t.device != dev
                              or not t.is_contiguous()):
            raise AssertionError(f"{name} must be contiguous ({D},) {dtype} or float32 on {dev}")
    if not 0 <= eps < math.inf:
        raise AssertionError(f"eps must be finite and not negative, got {eps}")
    if out is not None:
        if out.shape != q.shape or out.dtype != dtype or out.device != dev \
                or any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise AssertionError(f"out must be {tuple(q.shape)} {dtype} on {dev}, not expanded")
        same = out.data_ptr() == q.data_ptr() and out.stride() == q.stride()
        others = [k_pool, v_pool, positions, cos, sin, slots, q_norm, k_norm] + ([] if same else [q, k, v])
        if any(t is not None and overlap(out, t) for t in others):
            raise AssertionError("out must not share memory with the call's other tensors, but for q as it is")
    with on_stream(dev, stream):
        if any(s.data_ptr() % 16 for s in (cos, sin)) or (R // 2) % 4:
            cos, sin = cos.clone(), sin.clone()
        q, k, v = (_aligned(t) for t in (q, k, v))
        o = torch.empty((N, q.shape[1], D), device=dev, dtype=dtype) if out is None or not _is_aligned(out) else out
        qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), o.stride()
        nat.check(L.halo_rotate_rows(
            pool, q.data_ptr(), qs[0], qs[1], q.shape[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
            o.data_ptr(), os_[0], os_[1], N, positions.data_ptr(), positions.dtype == torch.int64, cos.data_ptr(),
            sin.data_ptr(), R // 2, cos.shape[0], R, interleaved, nat.ptr(q_norm),
            q_norm is not None and q_norm.dtype == torch.float32, nat.ptr(k_norm),
            k_norm is not None and k_norm.dtype == torch.float32, eps, slots.data_ptr(), nat.stream_ptr()),
            "halo_rotate_rows")
        if out is not None and o is not out:
            out.copy_(o)
    return o if out is None else out


def _is_aligned(t: torch.Tensor) -> bool:
    per = 16 // t.element_size()
    return t.stride(2) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) % per == 0 and t.stride(1) % per == 0


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t if _is_aligned(t) else t.clone(memory_format=torch.contiguous_format)
