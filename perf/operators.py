"""Performance cases of the block-pool operators: drafted token trees verified over a paged KV cache.

A case is a dict of plain values; ``kind`` names the operator:

  tables  blocks taken and given back for the requests' lengths, slots of their new rows (``update_block_tables``)
  append  new K/V rows written to their slots of the pool (``append_rows``)
  layout  ancestor masks and depths of the requests' drafted trees (``tree_layout``)
  attend  the drafted nodes attend the committed rows and their ancestors (``tree_attention``)
  commit  the rows of the accepted path moved behind the committed ones, all layers (``commit_path``)

Queries, keys and values are N(0, 1).  A pool is (blocks, H_kv, block rows, D), as a tier of ``TieredStorage``
keeps a layer; blocks are handed out in random order, as they are after a while of serving.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ESIZE = {"bf16": 2, "f16": 2, "f32": 4}
DEV = "cuda"


def listed():
    return [
        # a speculative step of a serving batch: every request gets room for its drafted rows
        dict(name="tables_step", kind="tables", B=16, bs=16, lo=8192, hi=131072, new=24, size_seed=3, fresh=False),
        # prompts of a full batch admitted at once
        dict(name="tables_prompts", kind="tables", B=256, bs=16, lo=128, hi=2048, new=0, size_seed=4, fresh=True),
        # one layer's drafted rows of a serving batch, where launches count
        dict(name="append_step", kind="append", L=1, N=203, H_kv=8, D=128, bs=16, blocks=512, dtype="bf16"),
        # one layer's rows of a 32k prompt
        dict(name="append_prompt", kind="append", L=1, N=32768, H_kv=8, D=128, bs=16, blocks=2304, dtype="bf16"),
        # the trees of a few chats
        dict(name="layout_step", kind="layout", B=4, nodes=16, size_seed=5),
        # wide trees of a full batch
        dict(name="layout_batch", kind="layout", B=256, nodes=200, size_seed=6),
        # one layer of a short chat turn with a small tree
        dict(name="attend_chat", kind="attend", B=1, H=32, H_kv=8, D=128, lo=4096, hi=4096, nodes=8, bs=16,
             dtype="bf16", size_seed=7, tree=True, lse=False),
        # one layer of a 32k context with a wide tree
        dict(name="attend_32k", kind="attend", B=1, H=32, H_kv=8, D=128, lo=32768, hi=32768, nodes=64, bs=16,
             dtype="bf16", size_seed=8, tree=True, lse=False),
        # a ragged serving batch of a 28/4-head model
        dict(name="attend_batch", kind="attend", B=16, H=28, H_kv=4, D=128, lo=1024, hi=32768, nodes=12, bs=32,
             dtype="f16", size_seed=9, tree=True, lse=True),
        # an fp32 model, blocks of 24 rows, partials to be merged with other chunks
        dict(name="attend_f32", kind="attend", B=3, H=16, H_kv=4, D=64, lo=300, hi=1500, nodes=9, bs=24,
             dtype="f32", size_seed=10, tree=True, lse=True),
        # the accepted path of one request, all layers
        dict(name="commit_step", kind="commit", B=1, L=32, H_kv=8, D=128, bs=16, lo=256, hi=256, path=5, nodes=32,
             dtype="bf16", size_seed=11),
        # the accepted paths of a serving batch of a 28/4-head model, all layers
        dict(name="commit_batch", kind="commit", B=32, L=28, H_kv=4, D=128, bs=16, lo=32, hi=256, path=8, nodes=48,
             dtype="f16", size_seed=12),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["tables", "append", "layout", "attend", "attend", "attend", "commit"])
    c = dict(kind=kind, size_seed=rng.randrange(10000))
    bs = rng.choice([8, 16, 16, 24, 32, 64])
    if kind == "tables":
        fresh = rng.random() < 0.4
        c.update(B=_log(rng, 1, 256), bs=bs, fresh=fresh, new=0 if fresh else rng.randint(1, 64))
        c.update(lo=rng.choice([1, 128]), hi=_log(rng, 256, 2048 if fresh else 32768))
    elif kind == "layout":
        c.update(B=_log(rng, 1, 256), nodes=_log(rng, 1, 200))
    else:
        H, H_kv = rng.choice([(32, 8), (28, 4), (16, 4), (8, 8)])
        c.update(H_kv=H_kv, D=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), bs=bs)
        if kind == "append":
            c.update(L=rng.choice([1, 1, 4]), N=_log(rng, 1, 8192))
            c.update(blocks=-(-c["N"] // bs) + rng.randint(1, 400))
        elif kind == "commit":
            path = rng.randint(1, 12)
            c.update(B=_log(rng, 1, 32), L=rng.randint(1, 28), lo=1, hi=_log(rng, 16, 256), path=path,
                     nodes=rng.randint(2 * path, 64))
        else:
            f32 = c["dtype"] == "f32"
            B = _log(rng, 1, 16)
            c.update(B=B, H=H, lo=rng.choice([1, 256]), hi=_log(rng, 512, 4096 if f32 else 32768), tree=rng.random() < 0.8,
                     nodes=_log(rng, 1, max(2, min(64, 192 // B))), lse=rng.choice([False, True]))
    return c


# ---------------------------------------------------------------- sizes

def _sizes(case):
    """Rows that each request holds and new (drafted) rows that it gets."""
    r = random.Random(case["size_seed"])
    B = case["B"]
    ctx = [_log(r, case["lo"], max(case["lo"], case["hi"])) for _ in range(B)]
    if case["kind"] == "tables":
        if case["fresh"]:
            return [0] * B, ctx
        return ctx, [r.randint(1, case["new"]) for _ in range(B)]
    if case["kind"] == "commit":
        return ctx, [r.randint(2 * case["path"], case["nodes"]) for _ in range(B)]
    return ctx, _nodes(case)


def _nodes(case):
    r = random.Random(case["size_seed"] + 1)
    n = case["nodes"]
    return [n] + [r.randint((n + 1) // 2, n) for _ in range(case["B"] - 1)]


def _width(case, ctx, new):
    """Columns of the block table: the longest request's blocks and a few spare ones."""
    return max(-(-(c + n) // case["bs"]) for c, n in zip(ctx, new)) + 3


def _parents(r: random.Random, n: int):
    """A drafted tree in breadth-first order: a root, then each node below one of the last few."""
    return [-1] + [r.randint(max(0, i // 2 - 2), max(0, i - 1 - i // 3)) for i in range(1, n)]


def _layout_of(case, seed):
    n = _nodes(case)
    r = random.Random(seed)
    return n, [p for k in n for p in _parents(r, k)]


def _path_moves(case, seed):
    """Accepted paths: the root, then nodes from behind the first ``path`` ones (so a row that is moved is never
    a row that another one moves to, and a pass can be repeated), and how many of them count."""
    ctx, n = _sizes(case)
    r = random.Random(seed)
    P = case["path"]
    paths = [[0] + sorted(r.sample(range(P, k), P - 1)) for k in n]
    return paths, [r.randint(max(1, P // 2), P) for _ in n]


# ---------------------------------------------------------------- inputs

def _gen(seed: int):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cu(n):
    t = [0]
    for k in n:
        t.append(t[-1] + k)
    return _i32(t)


def _tables(case, ctx, new, seed, spare):
    """A block table with the blocks of every request's ``ctx + new`` rows in random order, and what is left."""
    bs, W = case["bs"], _width(case, ctx, new)
    need = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    table = torch.full((case["B"], W), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table.to(DEV), order[at:].to(DEV), total


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = dict(kind=kind)
    if kind == "tables":
        ctx, new = _sizes(case)
        bs = case["bs"]
        own_blocks = [-(-c // bs) for c in ctx]
        spare = sum(-(-(c + n) // bs) for c, n in zip(ctx, new)) - sum(own_blocks) + 64
        table, free, total = _tables(case, ctx, [0] * len(ctx), seed, spare)
        W = _width(case, ctx, new)
        wide = torch.full((case["B"], W), -1, dtype=torch.int32, device=DEV)
        wide[:, :min(W, table.shape[1])] = table[:, :W]
        pad = torch.full((total,), -1, dtype=torch.int32, device=DEV)
        pad[:free.numel()] = free
        s.update(table=wide, n_blocks=_i32(own_blocks), free=pad, n_free=_i32([free.numel()]),
                 before=_i32(ctx), after=_i32([c + n for c, n in zip(ctx, new)]), bs=bs, max_rows=sum(new))
    elif kind == "append":
        dt = DTYPES[case["dtype"]]
        L, N, H, D, bs, P = (case[k] for k in ("L", "N", "H_kv", "D", "bs", "blocks"))
        lead = (L,) if L > 1 else ()
        slots = torch.randperm(P * bs, generator=torch.Generator().manual_seed(seed))[:N].sort().values
        blocks = torch.randperm(P, generator=torch.Generator().manual_seed(seed + 1))
        slots = (blocks[slots // bs] * bs + slots % bs).to(DEV)  # runs of rows in blocks of random order
        s.update(k_new=_randn(g, lead + (N, H, D), dt), v_new=_randn(g, lead + (N, H, D), dt), slots=slots,
                 k_pool=_randn(g, lead + (P, H, bs, D), dt), v_pool=_randn(g, lead + (P, H, bs, D), dt))
    elif kind == "layout":
        n, parents = _layout_of(case, seed)
        s.update(parents=_i32(parents), cu=_cu(n), max_nodes=max(n))
    elif kind == "attend":
        dt = DTYPES[case["dtype"]]
        ctx, n = _sizes(case)
        table, _, total = _tables(case, ctx, n, seed, 5)
        q = _randn(g, (sum(n), case["H"], case["D"]), dt)
        k = _randn(g, (total, case["H_kv"], case["bs"], case["D"]), dt)
        v = _randn(g, (total, case["H_kv"], case["bs"], case["D"]), dt)
        mask = None
        if case["tree"]:
            r = random.Random(seed)
            mask = torch.cat([_words(_parents(r, c), max(n)) for c in n]).to(DEV)
        s.update(q=q, k_pool=k, v_pool=v, table=table, lengths=_i32(ctx), cu=_cu(n), mask=mask, max_nodes=max(n),
                 longest=max(c + m for c, m in zip(ctx, n)), lse=case["lse"])
    else:
        dt = DTYPES[case["dtype"]]
        ctx, n = _sizes(case)
        table, _, total = _tables(case, ctx, n, seed, 2)
        shape = (case["L"], total, case["H_kv"], case["bs"], case["D"])
        paths, n_path = _path_moves(case, seed)
        s.update(k_pool=_randn(g, shape, dt), v_pool=_randn(g, shape, dt), table=table, lengths=_i32(ctx),
                 path=_i32(paths), n_path=_i32(n_path))
    return s


def _words(parents, max_nodes):
    """Ancestor bits (itself among them) of each node, 64 to an int64."""
    rows, W = [], (max_nodes + 63) // 64
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    cut = [[x >> 64 * w & (1 << 64) - 1 for w in range(W)] for x in rows]
    return torch.tensor([[x - (1 << 64) if x >> 63 else x for x in r] for r in cut], dtype=torch.int64)


# ---------------------------------------------------------------- one pass

def run(s):
    return {"tables": _run_tables, "append": _run_append, "layout": _run_layout, "attend": _run_attend,
            "commit": _run_commit}[s["kind"]](s)


def _run_tables(s):
    """Room for the new rows, and back: a step none of whose rows are kept leaves the tables as they were."""
    if own:
        import halo_amd
        a = (s["table"], s["n_blocks"], s["free"], s["n_free"])
        up = halo_amd.update_block_tables(*a, s["after"], s["before"], block_size=s["bs"], max_rows=s["max_rows"])
        halo_amd.update_block_tables(*a, s["before"], s["before"], block_size=s["bs"], max_rows=0)
        cu, slots, ok = up.cu_rows, up.slots, up.ok
    else:
        cu, slots, ok = _plain_tables(s, s["after"])
        _plain_tables(s, s["before"])
    return dict(cu=cu, slots=slots, ok=ok, table=s["table"], n_blocks=s["n_blocks"], free=s["free"],
                n_free=s["n_free"])


def _plain_tables(s, lengths):
    table, own_n, free, n_free, first, bs = (s[k] for k in ("table", "n_blocks", "free", "n_free", "before", "bs"))
    B, W = table.shape
    F = free.numel()
    need = (lengths + bs - 1) // bs
    col = torch.arange(W, device=DEV)[None, :]
    # surplus blocks, the last request's last block first, go on top of the free list
    back = ((col >= need[:, None]) & (col < own_n[:, None])).flip(0, 1).reshape(-1)
    rank = back.cumsum(0)
    to = torch.where(back, n_free + rank - 1, F)
    free_more = torch.cat([free, free[:1]])
    free_more.scatter_(0, to, table.flip(0, 1).reshape(-1))
    free.copy_(free_more[:F])
    n_free += rank[-1:]
    table.copy_(torch.where((col >= need[:, None]) & (col < own_n[:, None]), -1, table))
    # new blocks in the requests' order, while there are enough
    fits = need <= W
    grow = torch.where(fits, (need - own_n).clamp(min=0), 0)
    upto = grow.cumsum(0)
    ok = fits & ((grow == 0) | (upto <= n_free))
    take = (col >= own_n[:, None]) & (col < need[:, None]) & ok[:, None]
    at = n_free - 1 - ((upto - grow)[:, None] + col - own_n[:, None])
    table.copy_(torch.where(take, free[at.clamp(0, F - 1)], table))
    own_n.copy_(torch.where(ok, need, own_n))
    n_free -= (grow * ok).sum()
    # slots of the new rows, request after request
    cu = torch.cat([torch.zeros_like(need[:1]), (lengths - first).clamp(min=0).cumsum(0).int()])
    r = torch.arange(s["max_rows"], device=DEV)
    b = torch.searchsorted(cu[1:], r.int(), right=True).clamp(max=B - 1)
    p = r - cu[b] + first[b]
    slot = table[b, (p // bs).clamp(0, W - 1)].long() * bs + p % bs
    return cu, torch.where(ok[b] & (r < cu[-1]), slot, -1), ok


def _run_append(s):
    if own:
        import halo_amd
        halo_amd.append_rows(s["k_new"], s["v_new"], s["slots"], s["k_pool"], s["v_pool"])
    else:
        _plain_append(s["k_pool"], s["k_new"], s["slots"])
        _plain_append(s["v_pool"], s["v_new"], s["slots"])
    return dict(k=s["k_pool"], v=s["v_pool"])


def _plain_append(pool, new, slots):
    bs = pool.shape[-2]
    if pool.dim() == 5:
        pool[:, slots // bs, :, slots % bs] = new.transpose(0, 1)
    else:
        pool[slots // bs, :, slots % bs] = new


def _run_layout(s):
    if own:
        import halo_amd
        mask, depth = halo_amd.tree_layout(s["parents"], s["cu"], max_nodes=s["max_nodes"])
    else:
        mask, depth = _plain_layout(s["parents"], s["cu"], s["max_nodes"])
    return dict(mask=mask, depth=depth)


def _plain_layout(parents, cu, max_nodes):
    N, words = parents.numel(), (max_nodes + 63) // 64
    r = torch.arange(N, device=DEV)
    base = cu[torch.searchsorted(cu[1:], r.int(), right=True)].long()  # first node of each node's tree
    up = torch.where(parents >= 0, base + parents, N)  # N: above a root
    j = torch.arange(words * 64, device=DEV)
    bits = (r - base)[:, None] == j
    bits = torch.cat([bits, torch.zeros_like(bits[:1])])
    up = torch.cat([up, up.new_full((1,), N)])
    for _ in range((max_nodes - 1).bit_length()):  # ancestors at most 1, 3, 7, ... steps up
        bits = bits | bits[up]
        up = up[up]
    bits = bits[:N]
    mask = (bits.view(N, words, 64).long() << torch.arange(64, device=DEV)).sum(-1)
    return mask, (bits.sum(1) - 1).int()


def _run_attend(s):
    if own:
        import halo_amd
        got = halo_amd.tree_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lengths"], s["cu"],
                                      mask=s["mask"], max_nodes=s["max_nodes"], return_lse=s["lse"])
        return dict(out=got[0], lse=got[1]) if s["lse"] else dict(out=got)
    out, lse = _plain_attend(s)
    return dict(out=out, lse=lse) if s["lse"] else dict(out=out)


def _plain_attend(s):
    q, k_pool, v_pool, table, lengths, cu = (s[k] for k in ("q", "k_pool", "v_pool", "table", "lengths", "cu"))
    N, H, D = q.shape
    Hk, bs = k_pool.shape[1:3]
    B, M, T = table.shape[0], s["max_nodes"], s["longest"]
    node = torch.arange(M, device=DEV)
    pos = torch.arange(T, device=DEV)
    n = cu[1:] - cu[:-1]
    # every request's rows, and its nodes, in a padded batch
    block = table[:, pos // bs].long()
    there = (pos < (lengths + n)[:, None])[..., None, None]
    k = torch.where(there, k_pool[block.clamp(min=0), :, pos % bs].float(), 0)  # (B, T, Hk, D)
    v = torch.where(there, v_pool[block.clamp(min=0), :, pos % bs].float(), 0)
    row = (cu[:-1, None] + node).clamp(max=N - 1).long()
    qp = q[row].float().view(B, M, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    sc = (qp @ k.permute(0, 2, 3, 1)) * D ** -0.5  # (B, Hk, rep M, T)
    if s["mask"] is None:
        bits = (node[None, :] <= node[:, None]).expand(B, M, M)
    else:
        bits = (s["mask"][row][..., node // 64] >> node % 64 & 1).bool()
    at = (pos - lengths[:, None]).long()  # place among the nodes, negative for committed rows
    seen = bits.gather(2, at.clamp(0, M - 1)[:, None].expand(B, M, T))
    seen = (at < 0)[:, None] | (seen & (at < n[:, None])[:, None])
    sc = sc.view(B, Hk, H // Hk, M, T).masked_fill_(~seen[:, None, None], -torch.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -torch.inf, 0, top))
    den = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, -1, T) @ v.transpose(1, 2)).view(B, Hk, H // Hk, M, D) / torch.where(den > 0, den, 1)
    lse = (top + den.log()).squeeze(-1)
    # back to packed rows
    r = torch.arange(N, device=DEV)
    b = torch.searchsorted(cu[1:], r.int(), right=True)
    i = r - cu[b]
    return o[b, :, :, i].reshape(N, H, D).to(q.dtype), lse[b, :, :, i].reshape(N, H)


def _run_commit(s):
    if own:
        import halo_amd
        new = halo_amd.commit_path(s["k_pool"], s["v_pool"], s["table"], s["lengths"], s["path"], s["n_path"])
    else:
        new = _plain_commit(s["k_pool"], s["v_pool"], s["table"], s["lengths"], s["path"], s["n_path"])
    return dict(k=s["k_pool"], v=s["v_pool"], lengths=new)


def _plain_commit(k_pool, v_pool, table, lengths, path, n_path):
    bs, P = k_pool.shape[-2], path.shape[1]
    j = torch.arange(P, device=DEV)
    rises = torch.cat([path[:, :1] >= 0, path[:, 1:] > path[:, :-1]], 1)
    keep = rises.cumprod(1).bool() & (j < n_path[:, None])
    to = lengths[:, None] + j
    src = torch.where(keep, lengths[:, None] + path, to).long()  # a row that does not move is written as it is
    tb, sb = table.gather(1, to // bs).long(), table.gather(1, src // bs).long()
    k_pool[:, tb, :, to % bs] = k_pool[:, sb, :, src % bs]
    v_pool[:, tb, :, to % bs] = v_pool[:, sb, :, src % bs]
    return lengths + keep.sum(1).int()


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "tables":
        ctx, new = _sizes(case)
        bs = case["bs"]
        moved = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        # a block taken: its id read and entered; given back: the same; lengths and counts of both calls
        return dict(bytes=16 * moved + 8 * sum(new) + 2 * 16 * case["B"] + 5 * case["B"] + 4, flops=0)
    if kind == "append":
        row = case["H_kv"] * case["D"] * ESIZE[case["dtype"]]
        return dict(bytes=case["N"] * (8 + 4 * case["L"] * row), flops=0)
    if kind == "layout":
        n = _nodes(case)
        return dict(bytes=sum(n) * (4 + 8 * ((max(n) + 63) // 64) + 4) + 4 * len(n) + 4, flops=0)
    row = case["H_kv"] * case["D"] * ESIZE[case["dtype"]]
    ctx, n = _sizes(case)
    if kind == "attend":
        N, HD = sum(n), case["H"] * case["D"]
        rows = sum(ctx) + N
        io = 2 * N * HD * ESIZE[case["dtype"]] + (4 * N * case["H"] if case["lse"] else 0)
        tables = 4 * sum(-(-(c + k) // case["bs"]) for c, k in zip(ctx, n)) + 8 * case["B"]
        if case["tree"]:
            tables += 8 * N * ((max(n) + 63) // 64)
        seen = sum(k * c + (k if case["tree"] else k * (k + 1) // 2) for c, k in zip(ctx, n))
        return dict(bytes=2 * rows * row + io + tables, flops=4 * HD * seen)
    moved = case["B"] * 0.75 * case["path"]  # a path counts half of its nodes to all of them
    return dict(bytes=moved * case["L"] * row * 4 + case["B"] * (4 * case["path"] + 12), flops=0)


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "append": _exact_append, "layout": _exact_layout, "attend": _exact_attend,
            "commit": _exact_commit}[case["kind"]](case, seed, s)


def _exact_tables(case, seed, s):
    table, n, free, n_free, first = (s[k].tolist() for k in ("table", "n_blocks", "free", "n_free", "before"))
    bs, got = s["bs"], None
    for lengths in (s["after"].tolist(), first):
        need = [-(-x // bs) for x in lengths]
        stack = free[:n_free[0]]
        for b in reversed(range(len(n))):
            while n[b] > need[b]:
                n[b] -= 1
                stack.append(table[b][n[b]])
                table[b][n[b]] = -1
        ok, slots, cu, short = [], [], [0], False
        for b, k in enumerate(need):
            wants = k - n[b]
            fits = k <= len(table[b])
            short = short or (fits and wants > len(stack))
            ok.append(fits and not (wants > 0 and short))
            while ok[b] and n[b] < k:
                table[b][n[b]] = stack.pop()
                n[b] += 1
            rows = range(first[b], lengths[b])
            cu.append(cu[-1] + len(rows))
            slots += [table[b][p // bs] * bs + p % bs if ok[b] else -1 for p in rows]
        free[:max(n_free[0], len(stack))] = (stack + free[len(stack):])[:max(n_free[0], len(stack))]
        n_free = [len(stack)]
        if got is None:
            got = dict(cu=torch.tensor(cu, dtype=torch.int32), ok=torch.tensor(ok), slots=torch.tensor(slots))
    return dict(got, table=torch.tensor(table, dtype=torch.int32), n_blocks=torch.tensor(n, dtype=torch.int32),
                free=torch.tensor(free, dtype=torch.int32), n_free=torch.tensor(n_free, dtype=torch.int32))


def _exact_append(case, seed, s):
    got = {}
    for name in ("k", "v"):
        pool, new = s[name + "_pool"].double(), s[name + "_new"].double()
        rows = pool.transpose(-3, -2).reshape(*pool.shape[:-4], -1, case["H_kv"], case["D"])  # rows of all blocks
        rows.index_copy_(rows.dim() - 3, s["slots"], new)
        got[name] = rows.view(*pool.shape[:-3], case["bs"], case["H_kv"], case["D"]).transpose(-3, -2).contiguous()
    return got


def _exact_layout(case, seed, s):
    n, parents = _layout_of(case, seed)
    words, depth, at = [], [], 0
    for k in n:
        tree = parents[at:at + k]
        at += k
        words.append(_words(tree, max(n)))
        d = []
        for p in tree:
            d.append(d[p] + 1 if p >= 0 else 0)
        depth += d
    return dict(mask=torch.cat(words), depth=torch.tensor(depth, dtype=torch.int32))


def _exact_attend(case, seed, s):
    ctx, n = _sizes(case)
    H, Hk, D, bs = case["H"], case["H_kv"], case["D"], case["bs"]
    if 4 * H * D * sum(c * k for c, k in zip(ctx, n)) > 2e12:
        return None
    r = random.Random(seed)
    outs, lses, at = [], [], 0
    for b, (c, k) in enumerate(zip(ctx, n)):
        tree = _parents(r, k) if case["tree"] else range(-1, k - 1)
        sees = torch.zeros((k, c + k), dtype=torch.bool)
        sees[:, :c] = True
        for i in range(k):
            a = i
            while a >= 0:
                sees[i, c + a] = True
                a = tree[a]
        blocks = s["table"][b, :-(-(c + k) // bs)].long()
        kb = s["k_pool"][blocks].transpose(0, 1).reshape(Hk, -1, D)[:, :c + k]
        vb = s["v_pool"][blocks].transpose(0, 1).reshape(Hk, -1, D)[:, :c + k]
        qb = s["q"][at:at + k].double()
        at += k
        o, z = [], []
        for h in range(H):
            kh, vh = kb[h // (H // Hk)].double(), vb[h // (H // Hk)].double()
            sc = (qb[:, h] @ kh.T.contiguous() / math.sqrt(D)).masked_fill(~sees.to(DEV), -math.inf)
            z.append(torch.logsumexp(sc, 1))
            o.append(torch.softmax(sc, 1) @ vh)
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(z, 1))
    return dict(out=torch.cat(outs), lse=torch.cat(lses)) if case["lse"] else dict(out=torch.cat(outs))


def _exact_commit(case, seed, s):
    paths, n_path = _path_moves(case, seed)
    ctx, _ = _sizes(case)
    bs = case["bs"]
    table = s["table"].tolist()
    src, to = [], []
    for b, c in enumerate(ctx):
        for j, i in enumerate(paths[b][:n_path[b]]):
            src.append(table[b][(c + i) // bs] * bs + (c + i) % bs)
            to.append(table[b][(c + j) // bs] * bs + (c + j) % bs)
    got = {}
    for name in ("k", "v"):
        pool = s[name + "_pool"].double()
        rows = pool.transpose(2, 3).reshape(case["L"], -1, case["H_kv"], case["D"])
        kept = rows.clone()
        kept[:, to] = rows[:, src]
        got[name] = kept.view(case["L"], -1, bs, case["H_kv"], case["D"]).transpose(2, 3).contiguous()
    return dict(got, lengths=torch.tensor([c + k for c, k in zip(ctx, n_path)], dtype=torch.int32))
