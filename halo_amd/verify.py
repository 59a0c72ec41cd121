"""Verification of drafted trees: what of them the target model accepts.

The step between ``tree_attention`` and ``commit_path``: from the target's
probabilities behind every node, and given random numbers, the accepted path of
each request's tree and the token behind it, such that a request's tokens are
distributed as if the target had sampled them one by one.  The reference drafts
no tokens.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as nat
from . import block_pool as pool_calls
from .block_pool import _DTYPES, MAX_NODES, MAX_PATH, check_ints, on_stream


class Verified(NamedTuple):
    """What ``verify_tree`` found: ``path`` (B, max_path) int32, the accepted
    nodes, -1 behind them; ``n_path`` (B) int32, how many (0 for a request without
    nodes); ``token`` (B) int64, the token behind the path (-1 without nodes)."""

    path: torch.Tensor
    n_path: torch.Tensor
    token: torch.Tensor


def verify_tree(tokens: torch.Tensor, parents: torch.Tensor, cu_nodes: torch.Tensor, probs: torch.Tensor,
                accept: torch.Tensor, sample: torch.Tensor, *, max_nodes: int, draft_probs: Optional[torch.Tensor] = None,
                replacement: bool = True, max_path: Optional[int] = None, stream=None) -> Verified:
    """Nodes, ``parents`` (N) int32 and ``cu_nodes`` (B + 1) int32 as in
    ``tree_layout``: node 0 of a request is its last sampled token, which is always
    on the path, and other roots are not reached.  ``tokens`` (N) int64: the
    nodes' tokens; ``probs`` (N, V) bf16, fp16 or fp32: the target's
    probabilities behind each node; ``accept`` (N) and ``sample`` (B) fp32: random
    numbers in [0, 1).

    ``draft_probs`` (N, V), of the same dtype: the draft's probabilities that a
    node's children were drawn from, independently (``replacement``) or none twice;
    rows of nodes without children are not read.  Without them the children are
    taken as chosen (the draft's likeliest tokens, say).

    From node 0 on, the children of the node reached are tried in the order of
    their numbers.  With R what is left of the node's probabilities p, at first p,
    and Z = 1 at first, a child with token t drawn from q is accepted where
    ``accept * q[t] * Z < R[t]`` and the walk goes on from it; else R becomes
    ``max(R - Z q, 0)``, without t, and Z its sum.  Without draft probabilities a
    child is accepted where ``accept * Z < R[t]``; else t leaves R, and Z falls by
    ``p[t]`` (1 less the rejected tokens' p, also where p does not sum to 1, as
    rounded rows do not).  Where no child is accepted, or the path has ``max_path``
    (<= 64; default min(max_nodes, 64)) nodes, the next token is the first one at
    which the running sum of R exceeds ``sample`` times its whole (of p, should R
    be 0).

    ``max_nodes`` (<= 512) is the largest tree, further nodes are left out; V <=
    2^24.  Tokens outside [0, V) are not accepted; NaN and negative probabilities
    count as 0.  Sums are held in 64 bits, and equal calls give equal results."""
    if pool_calls.calls is not None and stream is None:
        r = pool_calls.calls.verify_tree(tokens, parents, cu_nodes, probs, accept, sample, max_nodes, draft_probs, replacement,
                                         min(max_nodes, MAX_PATH) if max_path is None else max_path)
        if r is not None:
            return Verified(*pool_calls.called(r, "halo_verify_tree"))
    L = nat.lib()
    dev = probs.device
    N, B = tokens.numel(), cu_nodes.numel() - 1
    if B < 1:
        raise AssertionError("cu_nodes needs an entry more than there are requests")
    if not 1 <= max_nodes <= MAX_NODES:
        raise AssertionError(f"max_nodes must be in [1, {MAX_NODES}], got {max_nodes}")
    if max_path is None:
        max_path = min(max_nodes, MAX_PATH)
    if not 1 <= max_path <= MAX_PATH:
        raise AssertionError(f"max_path must be in [1, {MAX_PATH}], got {max_path}")
    check_ints(tokens, "tokens", (N,), dev, torch.int64)
    check_ints(parents, "parents", (N,), dev)
    check_ints(cu_nodes, "cu_nodes", (B + 1,), dev)
    check_ints(accept, "accept", (N,), dev, torch.float32)
    check_ints(sample, "sample", (B,), dev, torch.float32)
    if probs.dtype not in _DTYPES or probs.dim() != 2 or probs.shape[0] != N or not 1 <= probs.shape[1] <= 1 << 24:
        raise AssertionError(f"probs must be ({N}, V <= 2^24) bf16, fp16 or fp32, got {probs.dtype} {tuple(probs.shape)}")
    V = probs.shape[1]
    if probs.stride(1) != 1 and V > 1:
        raise AssertionError("probs must have a unit last stride")
    if draft_probs is not None and (draft_probs.shape != probs.shape or draft_probs.dtype != probs.dtype
                                    or draft_probs.device != dev or (draft_probs.stride(1) != 1 and V > 1)):
        raise AssertionError(f"draft_probs must be {tuple(probs.shape)} {probs.dtype} on {dev} with unit last stride")
    with on_stream(dev, stream):
        path = torch.empty((B, max_path), device=dev, dtype=torch.int32)
        n_path = torch.empty(B, device=dev, dtype=torch.int32)
        token = torch.empty(B, device=dev, dtype=torch.int64)
        nat.check(L.halo_verify_tree(
            tokens.data_ptr(), parents.data_ptr(), cu_nodes.data_ptr(), B, N, max_nodes, V, nat.dtype_code(probs.dtype),
            probs.data_ptr(), probs.stride(0), nat.ptr(draft_probs), 0 if draft_probs is None else draft_probs.stride(0),
            replacement, accept.data_ptr(), sample.data_ptr(), max_path, path.data_ptr(), n_path.data_ptr(),
            token.data_ptr(), nat.stream_ptr()), "halo_verify_tree")
    return Verified(path, n_path, token)
