"""Block tables, drafted trees and attention over a paged cache, restated step
by step in Python and float64: no sums over prefixes, no tiles, no masks in
words."""
from __future__ import annotations

import math

import numpy as np


def update_block_tables(table, n_blocks, free, n_free, lengths, first, *, block_size, max_rows):
    """Lists in place of tensors; returns the changed state and (cu_rows, slots, ok)."""
    table = [list(r) for r in table]
    n_blocks, B, W = list(n_blocks), len(lengths), len(table[0])
    need = [-(-max(x, 0) // block_size) for x in lengths]
    cap = len(free)
    stack = list(free[:n_free])
    for b in reversed(range(B)):
        while n_blocks[b] > need[b]:
            n_blocks[b] -= 1
            stack.append(table[b][n_blocks[b]])
            table[b][n_blocks[b]] = -1
    stack = stack[:cap]
    rest = list(free)
    rest[:len(stack)] = stack
    ok, covered = [], True
    for b in range(B):
        wants = need[b] - n_blocks[b]
        if need[b] > W:
            ok.append(False)
            continue
        covered = covered and not wants > len(stack)
        ok.append(wants <= 0 or covered)
        while ok[b] and n_blocks[b] < need[b]:
            table[b][n_blocks[b]] = stack.pop()
            n_blocks[b] += 1
    cu, slots = [0], []
    for b in range(B):
        rows = range(max(first[b], 0), max(lengths[b], 0))
        cu.append(cu[-1] + len(rows))
        for p in rows:
            slots.append(table[b][p // block_size] * block_size + p % block_size if ok[b] else -1)
    slots = (slots + [-1] * max_rows)[:max_rows]
    return table, n_blocks, rest, len(stack), cu, slots, ok


def ancestors(parents):
    """For each node of a tree, the set of itself and its ancestors."""
    sets = []
    for i, p in enumerate(parents):
        sets.append({i} | (sets[p] if 0 <= p < i else set()))
    return sets


def words(sets, n_words):
    """The sets as int64 words, bit j % 64 of word j / 64."""
    out = np.zeros((len(sets), n_words), np.uint64)
    for i, s in enumerate(sets):
        for j in s:
            out[i, j // 64] |= np.uint64(1 << (j % 64))
    return out.view(np.int64)


def attend(q, k_pool, v_pool, table, lengths, cu, sees, scale):
    """q (N, H, D), pools (blocks, H_kv, rows, D) float64; ``sees[r]`` the tree
    rows that node r attends.  Returns out, lse, and for error bounds the
    weighted mean of |v| and the largest sum |q_d k_d| of an attended row."""
    N, H, D = q.shape
    P, Hk, bs, _ = k_pool.shape
    out, mean_abs = np.zeros((N, H, D)), np.zeros((N, H, D))
    lse, dots = np.full((N, H), -np.inf), np.zeros((N, H))
    for b in range(len(lengths)):
        for r in range(cu[b], cu[b + 1]):
            rows = list(range(lengths[b])) + [lengths[b] + j for j in sorted(sees[r])]
            at = [(table[b][p // bs], p % bs) for p in rows if p // bs < len(table[b])]
            at = [(x, y) for x, y in at if 0 <= x < P]
            if not at:
                continue
            blk, row = (np.array(x) for x in zip(*at))
            for h in range(H):
                k, v = k_pool[blk, h // (H // Hk), row], v_pool[blk, h // (H // Hk), row]
                with np.errstate(invalid="ignore"):
                    s = (k @ q[r, h]) * scale
                    m = s.max()
                    w = np.exp(s - m) if not math.isinf(m) else np.zeros_like(s)
                    den = w.sum()
                    if den == 0:
                        continue
                    lse[r, h] = m + np.log(den)
                    out[r, h] = (w[:, None] * v).sum(0) / den
                    mean_abs[r, h] = (w[:, None] * np.abs(v)).sum(0) / den
                    dots[r, h] = (np.abs(k) @ np.abs(q[r, h])).max() * scale
    return out, lse, mean_abs, dots
