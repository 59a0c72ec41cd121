"""Verified drafts, rotated rows, forked and compacted blocks, restated step by
step in Python and float64: distributions instead of one number for what is
left of them, sets of blocks instead of counts."""
from __future__ import annotations

import numpy as np


def verify(tokens, parents, cu, probs, accept, sample, *, max_nodes, draft=None, replacement=True, max_path):
    """Lists and float64 arrays (N, V); returns (path, n_path, token) as lists."""
    N, V = probs.shape
    paths, counts, last = [], [], []
    clean = lambda row: np.maximum(np.nan_to_num(row, nan=0.0, posinf=np.inf), 0.0)  # noqa: E731
    for b in range(len(cu) - 1):
        lo = max(cu[b], 0)
        n = max(min(cu[b + 1], N, lo + max_nodes) - lo, 0)
        if n == 0:
            paths.append([-1] * max_path)
            counts.append(0)
            last.append(-1)
            continue
        path = [0]
        while True:
            node = path[-1]
            rest, weight, rejected, found = clean(probs[lo + node]), 1.0, [], None
            q = clean(draft[lo + node]) if draft is not None else None
            for c in range(node + 1, n):
                t = tokens[lo + c]
                if len(path) >= max_path or parents[lo + c] != node or not 0 <= t < V:
                    continue
                if (q is None or not replacement) and (t in rejected or (q is not None and not q.sum() >= 0)):
                    continue
                if accept[lo + c] * (1.0 if q is None else q[t]) * weight < rest[t]:
                    found = c
                    break
                rejected.append(t)
                if q is None:
                    weight -= rest[t]
                    rest[t] = 0
                    continue
                rest = np.maximum(rest - weight * q, 0)
                rest[rejected] = 0
                weight = rest.sum()
                if not replacement:
                    left = 1 - q[t]
                    q[t] = 0
                    if not left > 0:
                        q[:] = np.nan  # nothing is left to draw
                    else:
                        q /= left
            if found is None:
                break
            path.append(found)
        if not rest.sum() > 0:
            rest = clean(probs[lo + path[-1]])
        upto = np.cumsum(rest)
        past = np.nonzero(upto > sample[b] * upto[-1])[0]
        there = np.nonzero(rest > 0)[0]
        last.append(int(past[0]) if len(past) else int(there[-1]) if len(there) else 0)
        counts.append(len(path))
        paths.append(path + [-1] * (max_path - len(path)))
    return paths, counts, last


def rotate(x, weight, eps, cos, sin, interleaved):
    """x (N, heads, D), cos and sin (N, R/2); returns the rotated heads and, for
    error bounds, |a c| + |b s| of each channel (|y| behind the rotated ones)."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight
    R = 2 * cos.shape[1]
    one = np.arange(0, R, 2) if interleaved else np.arange(R // 2)
    two = one + 1 if interleaved else one + R // 2
    c, s = cos[:, None], sin[:, None]
    out, size = y.copy(), np.abs(y)
    out[..., one] = y[..., one] * c - y[..., two] * s
    out[..., two] = y[..., two] * c + y[..., one] * s
    size[..., one] = np.abs(y[..., one] * c) + np.abs(y[..., two] * s)
    size[..., two] = np.abs(y[..., two] * c) + np.abs(y[..., one] * s)
    return out, size


def fork(table, n_blocks, free, n_free, shared, lengths, source, block_size, pools):
    """Lists (and arrays (L, blocks, H, rows, D) in ``pools``, changed in place);
    returns the changed state and (new_lengths, ok)."""
    B, W = len(source), len(table[0])
    held = [row[:min(max(n, 0), W)] for row, n in zip(table, n_blocks)]
    size = [min(max(x, 0), len(h) * block_size) for x, h in zip(lengths, held)]
    after, copies = [], []
    for b, a in enumerate(source):
        if not 0 <= a < B:
            after.append([])
            continue
        heir = a if source[a] == a else source.index(a)
        full, tail = divmod(size[a], block_size)
        if heir == b:
            after.append(list(held[a]))
        else:
            after.append(held[a][:full])
            if tail:
                copies.append((b, held[a][full], tail))
    count = lambda rows: {x: sum(r.count(x) for r in rows) for r in rows for x in r}  # noqa: E731
    has, had = count(after), count(held)
    freed = sorted(x for x in had if 0 <= x < len(shared) and x not in has)
    cap = len(free)
    stack = (list(free[:min(max(n_free, 0), cap)]) + freed)[:cap]
    if len(copies) > len(stack):
        return table, n_blocks, free, n_free, shared, list(lengths), False
    free = stack + list(free[len(stack):])
    for b, old, rows in copies:
        new = stack.pop()
        after[b].append(new)
        for pool in pools:
            pool[:, new, :, :rows] = pool[:, old, :, :rows]
    shared = list(shared)
    for x in set(had) | set(has):
        if 0 <= x < len(shared):
            shared[x] = max(has.get(x, 0) - 1, 0)
    table = [list(table[b]) if source[b] == b else after[b] + [-1] * (W - len(after[b])) for b in range(B)]
    return (table, [len(r) for r in after], free, len(stack), shared,
            [size[a] if 0 <= a < B else 0 for a in source], True)


def compact(table, n_blocks, free, n_free, shared, pools):
    """Returns the changed state and (new_id, n_used)."""
    P = len(shared)
    used = {x for row, n in zip(table, n_blocks) for x in row[:max(n, 0)] if 0 <= x < P}
    unused = {x for x in free[:min(max(n_free, 0), len(free))] if 0 <= x < P} - used
    places = sorted(used | unused)
    front, back = places[:len(used)], places[len(used):]
    moves = dict(zip(sorted(used & set(back)), sorted(unused & set(front))))
    shared = list(shared)
    for a, z in moves.items():
        for pool in pools:
            pool[:, z] = pool[:, a]
        shared[z], shared[a] = shared[a], 0
    stack = back[::-1]
    table = [[moves.get(x, x) if j < n else x for j, x in enumerate(row)] for row, n in zip(table, n_blocks)]
    return table, stack + list(free[len(stack):]), len(stack), shared, [moves.get(x, x) for x in range(P)], len(used)
