"""Performance cases of the operators around a paged KV cache: rows rotated into it, prompts attended in it, drafted
tokens verified, and its blocks forked, freed and compacted.

A case is a dict of plain values; ``kind`` names the operator:

  verify   the accepted path of each request's drafted tree, and the token behind it (``verify_tree``)
  rotate   heads of queries and keys normed and rotated, keys and values written to their slots (``rotate_rows``)
  fork     requests that go on with others' blocks, and requests that give theirs up (``fork_blocks``)
  compact  used blocks moved to the front of the pool (``compact_blocks``)
  chunk    new rows of prompts attend what their requests hold, and each other (``chunk_attention``)

Queries, keys and values are N(0, 1).  A pool is ([L,] blocks, H_kv, block rows, D), as a tier of ``TieredStorage``
keeps a layer, or all of them; blocks are handed out in random order, as they are after a while of serving.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ESIZE = {"bf16": 2, "f16": 2, "f32": 4}
DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # one chat with a small tree of the draft's likeliest tokens: launches and a chain of reads
        dict(name="verify_chat", kind="verify", B=1, V=32768, nodes=9, fan=3, draft="none", dtype="bf16", max_path=8,
             size_seed=21),
        # a serving batch, chains of sampled tokens
        dict(name="verify_chains", kind="verify", B=48, V=131072, nodes=8, fan=1, draft="with", dtype="f32", max_path=8,
             size_seed=22),
        # a batch of trees sampled without replacement, a vocabulary of odd size
        dict(name="verify_trees", kind="verify", B=13, V=50001, nodes=24, fan=4, draft="without", dtype="f32",
             max_path=12, size_seed=23),
        # a decode batch of an fp32 model: half of each head turned, neighbours as pairs, no norm
        dict(name="rotate_step", kind="rotate", N=27, H=16, H_kv=4, D=64, R=32, pairs=True, norm=False, bs=24, blocks=300,
             far=4096, dtype="f32"),
        # one layer's rows of a 32k prompt, heads normed
        dict(name="rotate_prompt", kind="rotate", N=32768, H=32, H_kv=8, D=128, R=128, pairs=False, norm=True, bs=16,
             blocks=2304, far=131072, dtype="bf16"),
        # beams of a few requests after a token, all layers of a 28/4-head model
        dict(name="fork_beams", kind="fork", B=32, beams=4, L=28, H_kv=4, D=128, bs=16, lo=256, hi=4096, dtype="bf16",
             size_seed=24, fresh=False),
        # many samples of a 16k prompt begun, and given up again
        dict(name="fork_samples", kind="fork", B=64, beams=64, L=8, H_kv=8, D=128, bs=16, lo=16383, hi=16383, dtype="bf16",
             size_seed=25, fresh=True),
        # a small pool's holes closed
        dict(name="compact_small", kind="compact", B=4, L=4, H_kv=4, D=64, bs=24, lo=100, hi=700, spare=50, dtype="f32",
             size_seed=26),
        # a pool of 2000 blocks, a third of them free
        dict(name="compact_large", kind="compact", B=24, L=8, H_kv=8, D=128, bs=16, lo=256, hi=2048, spare=700, dtype="f16",
             size_seed=27),
        # the end of a long prompt, one layer
        dict(name="chunk_tail", kind="chunk", B=1, H=32, H_kv=8, D=128, ctx_lo=32768, ctx_hi=32768, lo=601, hi=601, bs=16,
             dtype="bf16", size_seed=28, lse=False),
        # a prompt of 8192 rows at once, one layer
        dict(name="chunk_prompt", kind="chunk", B=1, H=32, H_kv=8, D=128, ctx_lo=0, ctx_hi=0, lo=8192, hi=8192, bs=16,
             dtype="bf16", size_seed=29, lse=False),
        # slices of prompts and single tokens of one batch of a 28/4-head model, partials to be merged
        dict(name="chunk_mixed", kind="chunk", B=9, H=28, H_kv=4, D=128, ctx_lo=1, ctx_hi=16384, lo=1, hi=2048, bs=32,
             dtype="f16", size_seed=30, lse=True),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))


def draw(rng: random.Random):
    kind = rng.choice(["verify", "verify", "rotate", "fork", "compact", "chunk", "chunk"])
    c = dict(kind=kind, size_seed=rng.randrange(10000))
    if kind == "verify":
        V = _log(rng, 200, 131072)
        nodes = _log(rng, 2, 64)
        c.update(V=V, nodes=nodes, B=_log(rng, 1, max(1, min(64, 40_000_000 // (V * nodes)))), fan=rng.randint(1, 5),
                 draft=rng.choice(["none", "with", "without"]), dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                 max_path=rng.randint(2, 16))
        return c
    H, H_kv = rng.choice([(32, 8), (28, 4), (16, 4), (8, 8)])
    c.update(H_kv=H_kv, D=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
             bs=rng.choice([8, 16, 16, 24, 32, 64]))
    if kind == "rotate":
        N = _log(rng, 1, 16384)
        c.update(H=H, N=N, R=rng.choice([c["D"], c["D"], c["D"] // 2, c["D"] // 4]), pairs=rng.random() < 0.3,
                 norm=rng.random() < 0.6, blocks=-(-N // c["bs"]) + rng.randint(1, 300), far=_log(rng, 64, 131072))
    elif kind == "fork":
        beams = rng.randint(2, 8)
        c.update(beams=beams, B=beams * rng.randint(1, 6), L=rng.randint(1, 12), lo=rng.choice([1, 128]),
                 hi=_log(rng, 128, 2048), fresh=rng.random() < 0.4)
    elif kind == "compact":
        c.update(B=_log(rng, 1, 24), L=rng.randint(1, 6), lo=1, hi=_log(rng, 16, 1024), spare=_log(rng, 1, 700))
    else:
        f32 = c["dtype"] == "f32"
        B = _log(rng, 1, 8)
        c.update(H=H, B=B, ctx_lo=rng.choice([0, 0, 300]), ctx_hi=_log(rng, 300, 2048 if f32 else 16384), lo=1,
                 hi=_log(rng, 1, 700 if f32 else max(2, 4096 // B)), lse=rng.random() < 0.5)
    return c


# ---------------------------------------------------------------- sizes

def _ctx(case, lo="lo", hi="hi"):
    """Rows that each request holds."""
    r = random.Random(case["size_seed"])
    if case["kind"] == "fork":  # beams of one request have grown together
        per = [_log(r, case["lo"], max(case["lo"], case["hi"])) for _ in range(case["B"] // case["beams"])]
        return [c for c in per for _ in range(case["beams"])]
    return [_log(r, case[lo], max(case[lo], case[hi])) if case[hi] else 0 for _ in range(case["B"])]


def _chunk_sizes(case):
    r = random.Random(case["size_seed"] + 1)
    ctx = _ctx(case, "ctx_lo", "ctx_hi")
    return ctx, [case["hi"]] + [_log(r, case["lo"], max(case["lo"], case["hi"])) for _ in ctx[1:]]


def _sources(case):
    """Whose blocks each row goes on with: beams picked within their request, or samples of its first row."""
    r = random.Random(case["size_seed"] + 2)
    b = case["beams"]
    if case["fresh"]:
        return [i // b * b for i in range(case["B"])]
    return [i // b * b + r.choice([0, 0, r.randrange(b)]) for i in range(case["B"])]


def _copies(case):
    """Rows of partly filled blocks that a fork copies."""
    ctx, src = _ctx(case), _sources(case)
    rows = 0
    for s in set(src):
        rows += (src.count(s) - 1) * (ctx[s] % case["bs"])
    return rows


def _tree_nodes(case):
    r = random.Random(case["size_seed"])
    n = case["nodes"]
    return [n] + [r.randint((n + 1) // 2, n) for _ in range(case["B"] - 1)]


def _tree(r: random.Random, n: int, fan: int):
    """Parents of a drafted tree: a root, then each node below an early one with less than ``fan`` children."""
    parents, count = [-1], [0]
    for i in range(1, n):
        free = [p for p in range(i) if count[p] < fan]
        p = free[min(len(free) - 1, int(len(free) * r.random() ** 2))]
        count[p] += 1
        parents.append(p)
        count.append(0)
    return parents


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


def _order(total, seed):
    return torch.randperm(total, generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def _tables(rows, bs, W, order):
    """Tables of requests with these rows, blocks in the given order, and how many of them are taken."""
    table = torch.full((len(rows), W), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(rows):
        k = -(-c // bs)
        table[b, :k] = order[at:at + k]
        at += k
    return table, at


def _meta(table, n_blocks, free, n_free, shared, lengths):
    """The tensors that a call changes, in one piece of memory, and a copy of it as it is before the call."""
    parts = [table, n_blocks, free, n_free, shared, lengths]
    flat = torch.cat([p.reshape(-1).int() for p in parts]).to(DEV)
    views, at = [], 0
    for p in parts:
        views.append(flat[at:at + p.numel()].view(p.shape))
        at += p.numel()
    return dict(zip(("table", "n_blocks", "free", "n_free", "shared", "lengths"), views), flat=flat, before=flat.clone())


def prepare(case, seed):
    return {"verify": _prepare_verify, "rotate": _prepare_rotate, "fork": _prepare_fork, "compact": _prepare_compact,
            "chunk": _prepare_chunk}[case["kind"]](case, seed)


def _prepare_verify(case, seed):
    g, r = _gen(seed), random.Random(seed)
    n, V, dt = _tree_nodes(case), case["V"], DTYPES[case["dtype"]]
    N = sum(n)
    parents = [p for k in n for p in _tree(r, k, case["fan"])]
    logits = torch.randn((N, V), generator=g, device=DEV) * 2.5
    probs = torch.softmax(logits, 1).to(dt)
    draft = torch.softmax(logits + 0.8 * torch.randn((N, V), generator=g, device=DEV), 1).to(dt)
    del logits
    # each node's children: the draft's likeliest tokens, or tokens drawn from it
    fan = min(case["fan"], V)
    if case["draft"] == "none":
        picks = draft.float().topk(fan).indices
    elif case["draft"] == "with":
        picks = torch.multinomial(draft.float(), fan, replacement=True, generator=g)
    else:
        gumbel = -torch.log(torch.empty((N, V), device=DEV).exponential_(generator=g))
        picks = (draft.float().log() + gumbel).topk(fan).indices
    where, which, at = [], [], 0
    for k in n:
        seen = [0] * k
        for p in parents[at:at + k]:
            where.append(at + max(p, 0))
            which.append(seen[p] if p >= 0 else 0)
            if p >= 0:
                seen[p] += 1
        at += k
    tokens = picks[torch.tensor(where, device=DEV), torch.tensor(which, device=DEV)]
    return dict(kind="verify", tokens=tokens, parents=_i32(parents), cu=_cu(n), probs=probs,
                draft=None if case["draft"] == "none" else draft, replace=case["draft"] != "without", max_nodes=max(n),
                max_path=case["max_path"], accept=torch.rand(N, generator=g, device=DEV),
                sample=torch.rand(case["B"], generator=g, device=DEV))


def _prepare_rotate(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    N, H, Hk, D, R, bs, P = (case[k] for k in ("N", "H", "H_kv", "D", "R", "bs", "blocks"))
    qkv = _randn(g, (N, H + 2 * Hk, D), dt)  # one projection's rows
    slots = torch.randperm(P * bs, generator=torch.Generator().manual_seed(seed))[:N].sort().values
    slots = (_order(P, seed + 1).long()[slots // bs] * bs + slots % bs).to(DEV)  # runs of rows in blocks of random order
    far = case["far"]
    angle = torch.arange(far, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    first = int(torch.randint(0, max(1, far - N), (1,), generator=torch.Generator().manual_seed(seed)))
    weights = [(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dt) for _ in range(2)]
    return dict(kind="rotate", q=qkv[:, :H], k=qkv[:, H:H + Hk], v=qkv[:, H + Hk:],
                positions=(first + torch.arange(N, device=DEV)) % far, cos=angle.cos().float(), sin=angle.sin().float(),
                q_norm=weights[0] if case["norm"] else None, k_norm=weights[1] if case["norm"] else None,
                pairs=case["pairs"], slots=slots, k_pool=_randn(g, (P, Hk, bs, D), dt), v_pool=_randn(g, (P, Hk, bs, D), dt))


def _prepare_fork(case, seed):
    g, dt, bs, beams = _gen(seed), DTYPES[case["dtype"]], case["bs"], case["beams"]
    ctx, src = _ctx(case), _sources(case)
    B, W = case["B"], max(-(-c // bs) for c in ctx) + 2
    full, tails = [c // bs for c in ctx], [int(c % bs > 0) for c in ctx]
    total = sum(full[::beams]) + sum(tails) + B + 3
    order = _order(total, seed)
    table, shared, at = torch.full((B, W), -1, dtype=torch.int32), torch.zeros(total, dtype=torch.int32), 0
    n_blocks = [0] * B
    for b in range(B):
        if case["fresh"] and b % beams:
            continue
        if b % beams == 0:
            lead = order[at:at + full[b]]
            at += full[b]
            shared[lead.long()] = 0 if case["fresh"] else beams - 1
        table[b, :full[b]] = lead
        table[b, full[b]:full[b] + tails[b]] = order[at:at + tails[b]]
        at += tails[b]
        n_blocks[b] = full[b] + tails[b]
    free = torch.full((total,), -1, dtype=torch.int32)
    free[:total - at] = order[at:]
    lengths = [c if n else 0 for c, n in zip(ctx, n_blocks)]
    shape = (case["L"], total, case["H_kv"], bs, case["D"])
    drop = [b if b % beams == 0 else -1 for b in range(B)]
    return dict(_meta(table, torch.tensor(n_blocks), free, torch.tensor([total - at]), shared, torch.tensor(lengths)),
                kind="fork", bs=bs, source=_i32(src), drop=_i32(drop) if case["fresh"] else None,
                k_pool=_randn(g, shape, dt), v_pool=_randn(g, shape, dt))


def _prepare_compact(case, seed):
    g, dt, bs = _gen(seed), DTYPES[case["dtype"]], case["bs"]
    ctx = _ctx(case)
    W = max(-(-c // bs) for c in ctx) + 2
    n_blocks = [-(-c // bs) for c in ctx]
    total = sum(n_blocks) + case["spare"]
    order = _order(total, seed)
    table, at = _tables(ctx, bs, W, order)
    free = torch.full((total,), -1, dtype=torch.int32)
    free[:total - at] = order[at:]
    shape = (case["L"], total, case["H_kv"], bs, case["D"])
    return dict(_meta(table, torch.tensor(n_blocks), free, torch.tensor([total - at]), torch.zeros(total), torch.tensor(ctx)),
                kind="compact", k_pool=_randn(g, shape, dt), v_pool=_randn(g, shape, dt))


def _prepare_chunk(case, seed):
    g, dt, bs = _gen(seed), DTYPES[case["dtype"]], case["bs"]
    ctx, n = _chunk_sizes(case)
    rows = [c + k for c, k in zip(ctx, n)]
    W = max(-(-c // bs) for c in rows) + 3
    total = sum(-(-c // bs) for c in rows) + 5
    table, _ = _tables(rows, bs, W, _order(total, seed))
    shape = (total, case["H_kv"], bs, case["D"])
    return dict(kind="chunk", q=_randn(g, (sum(n), case["H"], case["D"]), dt), k_pool=_randn(g, shape, dt),
                v_pool=_randn(g, shape, dt), table=table.to(DEV), lengths=_i32(ctx), cu=_cu(n), max_rows=max(n),
                sizes=(ctx, n), lse=case["lse"])


# ---------------------------------------------------------------- one pass

def run(s):
    return {"verify": _run_verify, "rotate": _run_rotate, "fork": _run_fork, "compact": _run_compact,
            "chunk": _run_chunk}[s["kind"]](s)


def _run_verify(s):
    if own:
        import halo_amd
        got = halo_amd.verify_tree(s["tokens"], s["parents"], s["cu"], s["probs"], s["accept"], s["sample"],
                                   max_nodes=s["max_nodes"], draft_probs=s["draft"], replacement=s["replace"],
                                   max_path=s["max_path"])
        return dict(path=got.path, n_path=got.n_path, token=got.token)
    path, n_path, token = _plain_verify(s)
    return dict(path=path, n_path=n_path, token=token)


def _plain_verify(s):
    tokens, parents, cu, probs, draft, replace = (s[k] for k in ("tokens", "parents", "cu", "probs", "draft", "replace"))
    N, V = probs.shape
    lo, n = cu[:-1].long(), cu[1:] - cu[:-1]
    B, P = n.numel(), s["max_path"]
    each = torch.arange(B, device=DEV)
    f64 = dict(dtype=torch.float64, device=DEV)
    at = torch.zeros(B, dtype=torch.int32, device=DEV)  # the node reached
    path = torch.full((B, P), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    n_path = torch.ones(B, dtype=torch.int32, device=DEV)
    gone = torch.zeros((B, V), dtype=torch.bool, device=DEV)  # tokens rejected there
    S, Z, Q = torch.zeros(B, **f64), torch.ones(B, **f64), torch.zeros(B, **f64)

    def left():  # what is left of the target's probabilities
        rest = probs[lo + at].double()
        if draft is not None:
            rest = (rest - S[:, None] * draft[lo + at].double()).clamp(min=0)
        return rest.masked_fill(gone, 0)

    for i in range(1, s["max_nodes"]):  # a node's children lie behind it, so one walk over the nodes tries them in turn
        row = (lo + i).clamp(max=N - 1)
        t = tokens[row]
        was = gone[each, t]
        p = probs[lo + at, t].double()
        q = draft[lo + at, t].double() if draft is not None else torch.ones(B, **f64)
        tried = (i < n) & (parents[row] == at) & (n_path < P)
        if draft is None or not replace:
            tried = tried & ~was & (1 - Q > 0)
        d = 1 / (1 - Q) if draft is not None and not replace else torch.ones(B, **f64)
        r = p - S * q if draft is not None else p
        r = torch.where(was, 0, r.clamp(min=0))
        yes = tried & (s["accept"][row].double() * q * d * Z < r)
        no = tried & ~yes
        gone[each, t] = was | no
        if draft is not None:
            S = torch.where(no, S + Z * d, S)
            if not replace:
                Q = torch.where(no, Q + q, Q)
            Z = torch.where(no, left().sum(1), Z)
        else:
            Z = torch.where(no, Z - p, Z)
        # on to the accepted child
        path.scatter_(1, n_path.clamp(max=P - 1)[:, None].long(),
                      torch.where(yes, i, path.gather(1, n_path.clamp(max=P - 1)[:, None].long())[:, 0])[:, None].int())
        n_path = n_path + yes
        at = torch.where(yes, i, at).int()
        gone &= ~yes[:, None]
        S, Z, Q = torch.where(yes, 0, S), torch.where(yes, 1, Z), torch.where(yes, 0, Q)
    rest = left()
    total = rest.sum(1, keepdim=True)
    rest = torch.where(total > 0, rest, probs[lo + at].double())
    upto = rest.cumsum(1)
    token = (upto <= s["sample"].double()[:, None] * upto[:, -1:]).sum(1)
    last = torch.where(rest > 0, torch.arange(V, device=DEV), 0).amax(1)
    return path, n_path, torch.minimum(token, last)


def _run_rotate(s):
    if own:
        import halo_amd
        q = halo_amd.rotate_rows(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], s["slots"], s["k_pool"],
                                 s["v_pool"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, interleaved=s["pairs"])
    else:
        bs = s["k_pool"].shape[-2]
        q = _plain_rotate(s, s["q"], s["q_norm"])
        s["k_pool"][s["slots"] // bs, :, s["slots"] % bs] = _plain_rotate(s, s["k"], s["k_norm"])
        s["v_pool"][s["slots"] // bs, :, s["slots"] % bs] = s["v"]
    return dict(q=q, k=s["k_pool"], v=s["v_pool"])


def _plain_rotate(s, x, weight):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    R = 2 * cos.shape[-1]
    turned = y.clone()
    if s["pairs"]:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned[..., 0:R:2] = a * cos - b * sin
        turned[..., 1:R:2] = b * cos + a * sin
    else:
        a, b = y[..., :R // 2], y[..., R // 2:R]
        turned[..., :R // 2] = a * cos - b * sin
        turned[..., R // 2:R] = b * cos + a * sin
    return turned.to(x.dtype)


def _run_fork(s):
    """Beams go on (the same choice again and again); or samples begin and end, which leaves the tables as they were."""
    oks = []
    lengths = s["lengths"]
    for source in (s["source"], s["drop"]):
        if source is None:
            continue
        if own:
            import halo_amd
            lengths, ok = halo_amd.fork_blocks(s["table"], s["n_blocks"], s["free"], s["n_free"], s["shared"], lengths,
                                               source, s["k_pool"], s["v_pool"])
        else:
            lengths, ok = _plain_fork(s, lengths, source)
        oks.append(ok)
    return dict(table=s["table"], n_blocks=s["n_blocks"], free=s["free"], n_free=s["n_free"], shared=s["shared"],
                lengths=lengths, ok=torch.cat(oks), k=s["k_pool"], v=s["v_pool"])


def _plain_fork(s, lengths, source):
    table, own_n, free, n_free, shared, bs = (s[k] for k in ("table", "n_blocks", "free", "n_free", "shared", "bs"))
    B, W = table.shape
    F, X = free.numel(), shared.numel()
    row, col = torch.arange(B, device=DEV), torch.arange(W, device=DEV)[None, :]
    src = source.long()
    lives = src >= 0
    src = src.clamp(min=0)
    full = lengths // bs
    count = torch.zeros_like(own_n).index_add_(0, src, lives.int())
    first = torch.where(lives[None, :] & (src[None, :] == row[:, None]), row, B).amin(1)  # each row's first follower
    heir = torch.where(lives & (src == row), row, B)  # it stays its own, or the first follower has it
    heir = torch.where(heir < B, heir, first)
    is_heir = lives & (heir[src] == row)
    # holders that each block gains and loses; blocks without any are free, the lowest first
    gain = torch.where(col < full[:, None], count[:, None] - 1, (count > 0).int()[:, None] - 1)
    gain = torch.where(col < own_n[:, None], gain, 0).int()
    change = torch.zeros(X + 1, dtype=torch.int32, device=DEV)
    change.index_add_(0, torch.where(col < own_n[:, None], table, X).reshape(-1).long(), gain.reshape(-1))
    change = change[:X]
    freed = (change < 0) & (shared + 1 + change == 0)
    rank = freed.int().cumsum(0)
    wants = lives & ~is_heir & (lengths[src] % bs > 0)
    nth = wants.int().cumsum(0)
    ok = n_free + rank[-1:] >= nth[-1:]
    stack = torch.cat([free, free[:1]])
    stack.scatter_(0, torch.where(freed, n_free + rank - 1, F).long().clamp(max=F), torch.arange(X, device=DEV).int())
    top = n_free + rank[-1:]
    fresh = stack[(top - nth).clamp(0, F - 1).long()]
    keep = torch.where(is_heir[:, None], own_n[src][:, None], full[src][:, None])
    new = torch.where(lives[:, None] & (col < keep), table[src], -1)
    new = torch.where(wants[:, None] & (col == full[src][:, None]), fresh[:, None], new)
    new = torch.where((lives & (src == row))[:, None], table, new)
    # rows of the partly filled blocks
    line = torch.arange(bs, device=DEV)
    tail = table[src, full[src].clamp(max=W - 1).long()].clamp(min=0).long()
    moves = (ok & wants)[:, None] & (line < (lengths[src] % bs)[:, None])
    to = torch.where(wants, fresh, tail).long()
    for pool in (s["k_pool"], s["v_pool"]):
        # (rows that stay are written as they are, one after another, so that none is lost among equal places)
        for b in range(B):
            old = pool[:, tail[b:b + 1]]
            pool[:, to[b:b + 1]] = torch.where(moves[b][:, None], old, pool[:, to[b:b + 1]])
    n_new = torch.where(lives, torch.where(is_heir, own_n[src], full[src] + wants.int()), 0).int()
    table.copy_(torch.where(ok, new, table))
    free.copy_(torch.where(ok, stack[:F], free))
    own_n.copy_(torch.where(ok, n_new, own_n))
    n_free.copy_(torch.where(ok, top - nth[-1:], n_free))
    shared.copy_(torch.where(ok, torch.where(freed, 0, shared + change), shared))
    return torch.where(ok, torch.where(lives, lengths[src], 0), lengths).int(), ok


def _run_compact(s):
    """Starts from the same tables in every pass."""
    s["flat"].copy_(s["before"])
    if own:
        import halo_amd
        new_id, n_used = halo_amd.compact_blocks(s["table"], s["n_blocks"], s["free"], s["n_free"], s["shared"], s["k_pool"],
                                                 s["v_pool"])
    else:
        new_id, n_used = _plain_compact(s)
    return dict(table=s["table"], free=s["free"], n_free=s["n_free"], shared=s["shared"], new_id=new_id, n_used=n_used,
                k=s["k_pool"], v=s["v_pool"])


def _plain_compact(s):
    table, own_n, free, n_free, shared = (s[k] for k in ("table", "n_blocks", "free", "n_free", "shared"))
    B, W = table.shape
    F, X = free.numel(), shared.numel()
    held = torch.arange(W, device=DEV)[None, :] < own_n[:, None]
    place = torch.arange(F, device=DEV)
    flag = torch.zeros(X + 1, dtype=torch.int32, device=DEV)
    flag[torch.where(place < n_free, free, X).long()] = 2
    flag[torch.where(held, table, X).reshape(-1).long()] = 1
    flag = flag[:X]
    used, there = flag == 1, flag > 0
    n_used = used.sum().int()[None]
    nth = there.int().cumsum(0)  # the pool's n-th block of those that are used or free
    front = there & (nth <= n_used)
    gap, move = front & ~used, used & ~front
    nth_gap, nth_move = gap.int().cumsum(0), move.int().cumsum(0)
    ids = torch.arange(X, device=DEV)
    gaps = torch.zeros(X + 1, dtype=torch.int64, device=DEV).scatter_(0, torch.where(gap, nth_gap - 1, X).long(), ids)
    new_id = torch.where(move, gaps[(nth_move - 1).clamp(min=0).long()], ids)
    for pool in (s["k_pool"], s["v_pool"]):
        old = pool.index_select(1, torch.where(gap, 0, ids))  # all blocks, each at its old place
        take = ids.clone()
        take = torch.cat([take, take[:1]]).scatter_(0, torch.where(move, new_id, X), ids)[:X]
        pool.copy_(torch.where(gap[:, None, None, None], old.index_select(1, take), pool))
    table.copy_(torch.where(held, new_id[table.clamp(min=0).long()].int(), table))
    gone = move.int()
    moved = torch.zeros(X + 1, dtype=torch.int32, device=DEV)
    moved.scatter_(0, torch.where(move, new_id, X), shared)
    shared.copy_(torch.where(gap, moved[:X], torch.where(gone > 0, 0, shared)))
    # the lowest free block on top
    back = there & ~front
    total = nth[-1:] - n_used
    at = torch.where(back, total - (nth - n_used), F)
    stack = torch.cat([free, free[:1]])
    stack.scatter_(0, at.long(), ids.int())
    free.copy_(stack[:F])
    n_free.copy_(total)
    return new_id.int(), n_used


def _run_chunk(s):
    if own:
        import halo_amd
        got = halo_amd.chunk_attention(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lengths"], s["cu"],
                                       max_rows=s["max_rows"], return_lse=s["lse"])
        return dict(out=got[0], lse=got[1]) if s["lse"] else dict(out=got)
    out, lse = _plain_chunk(s)
    return dict(out=out, lse=lse) if s["lse"] else dict(out=out)


def _plain_chunk(s):
    q, k_pool, v_pool, table = (s[k] for k in ("q", "k_pool", "v_pool", "table"))
    N, H, D = q.shape
    Hk, bs = k_pool.shape[1:3]
    out, lse = torch.empty_like(q), torch.empty((N, H), device=DEV)
    at = 0
    for b, (c, n) in enumerate(zip(*s["sizes"])):
        blocks = table[b, :-(-(c + n) // bs)].long()
        k = k_pool[blocks].transpose(0, 1).reshape(Hk, -1, D)[:, :c + n].float()
        v = v_pool[blocks].transpose(0, 1).reshape(Hk, -1, D)[:, :c + n].float()
        kt = k.transpose(1, 2).contiguous()
        for i in range(0, n, 1024):  # what a block of rows may see, and no more
            m = min(1024, n - i)
            T = c + i + m
            qb = q[at + i:at + i + m].float().view(m, Hk, -1, D).permute(1, 2, 0, 3).reshape(Hk, -1, D)
            sc = (qb @ kt[:, :, :T]).view(Hk, -1, m, T) * D ** -0.5
            pos = torch.arange(T, device=DEV)
            sc.masked_fill_(pos[None, :] > c + i + torch.arange(m, device=DEV)[:, None], -torch.inf)
            top = sc.amax(-1, keepdim=True)
            p = torch.exp(sc - top)
            den = p.sum(-1, keepdim=True)
            o = (p.view(Hk, -1, T) @ v[:, :T]).view(Hk, -1, m, D) / den
            out[at + i:at + i + m] = o.permute(2, 0, 1, 3).reshape(m, H, D)
            lse[at + i:at + i + m] = (top + den.log()).squeeze(-1).permute(2, 0, 1).reshape(m, H)
        at += n
    return out, lse


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "verify":
        # one row of the target's probabilities a request, the draft's too where a child was rejected (about half)
        rows = case["B"] * (1.5 if case["draft"] != "none" else 1)
        return dict(bytes=rows * case["V"] * ESIZE[case["dtype"]] + 24 * sum(_tree_nodes(case)), flops=3 * rows * case["V"])
    row = case["H_kv"] * case["D"] * ESIZE[case["dtype"]]
    if kind == "rotate":
        q = case["H"] * case["D"] * ESIZE[case["dtype"]]
        return dict(bytes=case["N"] * (2 * q + 4 * row + 4 * case["R"] + 16),
                    flops=case["N"] * (case["H"] + case["H_kv"]) * (3 * case["R"] + 4 * case["D"] * case["norm"]))
    if kind == "fork":
        entries = sum(-(-c // case["bs"]) for c in _ctx(case))
        return dict(bytes=4 * _copies(case) * case["L"] * row + 8 * entries, flops=0)
    if kind == "compact":
        used = sum(-(-c // case["bs"]) for c in _ctx(case))
        moved = used * case["spare"] / (used + case["spare"])  # used blocks among the last ``spare`` of the pool
        return dict(bytes=4 * moved * case["bs"] * case["L"] * row + 8 * (used + case["spare"]), flops=0)
    ctx, n = _chunk_sizes(case)
    HD = case["H"] * case["D"]
    io = 2 * sum(n) * HD * ESIZE[case["dtype"]] + (4 * sum(n) * case["H"] if case["lse"] else 0)
    pairs = sum(k * c + k * (k + 1) // 2 for c, k in zip(ctx, n))
    return dict(bytes=2 * (sum(ctx) + sum(n)) * row + io, flops=4 * HD * pairs)


# ---------------------------------------------------------------- from the definitions, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"verify": _exact_verify, "rotate": _exact_rotate, "fork": _exact_fork, "compact": _exact_compact,
            "chunk": _exact_chunk}[case["kind"]](case, s)


def _exact_verify(case, s):
    cu, parents, tokens = s["cu"].tolist(), s["parents"].tolist(), s["tokens"].tolist()
    accept, sample = s["accept"].tolist(), s["sample"].tolist()
    paths, counts, last = [], [], []
    for b in range(case["B"]):
        lo, n = cu[b], cu[b + 1] - cu[b]
        path = [0]
        while True:
            node = path[-1]
            rest = s["probs"][lo + node].double()  # the target's distribution, then what is left of it
            q = s["draft"][lo + node].double() if s["draft"] is not None else None
            weight, found, seen = 1.0, None, set()
            for c in range(node + 1, n if len(path) < case["max_path"] else 0):
                if parents[lo + c] != node:
                    continue
                t = tokens[lo + c]
                if q is None:
                    if t in seen:
                        continue
                    if accept[lo + c] * weight < float(rest[t]):
                        found = c
                        break
                    weight -= float(rest[t])
                    rest = rest.clone()
                    rest[t] = 0
                else:
                    if accept[lo + c] * float(q[t]) * weight < float(rest[t]):
                        found = c
                        break
                    rest = torch.clamp(rest - weight * q, min=0)
                    rest[t] = 0
                    weight = float(rest.sum())
                    if case["draft"] == "without":
                        q = q.clone()
                        gone, q[t] = float(q[t]), 0
                        q = q / (1 - gone)
                seen.add(t)
            if found is None:
                break
            path.append(found)
        if not float(rest.sum()) > 0:
            rest = s["probs"][lo + path[-1]].double()
        upto = rest.cumsum(0)
        t = int((upto <= sample[b] * float(upto[-1])).sum())
        last.append(min(t, int(torch.nonzero(rest)[-1])))
        counts.append(len(path))
        paths.append(path + [-1] * (case["max_path"] - len(path)))
    return dict(path=torch.tensor(paths, dtype=torch.int32), n_path=torch.tensor(counts, dtype=torch.int32),
                token=torch.tensor(last))


def _exact_rotate(case, s):
    N, D, R, bs = case["N"], case["D"], case["R"], case["bs"]
    cos, sin = (s[k].double()[s["positions"]].unsqueeze(1) for k in ("cos", "sin"))
    one = [2 * i if case["pairs"] else i for i in range(R // 2)]
    two = [2 * i + 1 if case["pairs"] else i + R // 2 for i in range(R // 2)]

    def turn(x, weight):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * weight.double()
        z = torch.complex(x[..., one], x[..., two]) * torch.complex(cos, sin)
        x = x.clone()
        x[..., one], x[..., two] = z.real, z.imag
        return x

    got = dict(q=turn(s["q"], s["q_norm"]))
    for name, new in (("k", turn(s["k"], s["k_norm"])), ("v", s["v"].double())):
        rows = s[name + "_pool"].double().transpose(1, 2).reshape(-1, case["H_kv"], D)
        rows.index_copy_(0, s["slots"], new)
        got[name] = rows.view(-1, bs, case["H_kv"], D).transpose(1, 2).contiguous()
    return got


def _exact_fork(case, s):
    bs = case["bs"]
    table, n, free, shared, length = (s[k].tolist() for k in ("table", "n_blocks", "free", "shared", "lengths"))
    cap, stack, oks = len(free), free[:int(s["n_free"])], []
    pools = {name: s[name + "_pool"].double() for name in ("k", "v")}
    W = s["table"].shape[1]
    for source in [s["source"].tolist()] + ([s["drop"].tolist()] if s["drop"] is not None else []):
        held = [row[:k] for row, k in zip(table, n)]
        after, copies = [], []
        for b, a in enumerate(source):
            if a < 0:
                after.append([])
                continue
            heir = a if source[a] == a else source.index(a)
            full, tail = divmod(length[a], bs)
            after.append(held[a] if heir == b else held[a][:full] + [None] * (tail > 0))
            if heir != b and tail:
                copies.append((b, full, held[a][full], tail))
        holders = {}
        for row in after:
            for x in row:
                holders[x] = holders.get(x, 0) + 1
        freed = sorted({x for row in held for x in row if x not in holders})
        ok = len(stack) + len(freed) >= len(copies)
        oks.append(ok)
        if not ok:
            continue
        stack += freed
        free[:len(stack)] = stack
        for b, at, old, rows in copies:
            new = stack.pop()
            after[b] = after[b][:at] + [new]
            holders[new] = 1
            for pool in pools.values():
                pool[:, new, :, :rows] = pool[:, old, :, :rows]
        shared = [holders.get(x, 1) - 1 for x in range(len(shared))]
        n = [len(row) for row in after]
        table = [row + [-1] * (W - len(row)) for row in after]
        length = [length[a] if a >= 0 else 0 for a in source]
    i32 = dict(dtype=torch.int32)
    return dict(table=torch.tensor(table, **i32), n_blocks=torch.tensor(n, **i32), free=torch.tensor(free[:cap], **i32),
                n_free=torch.tensor([len(stack)], **i32), shared=torch.tensor(shared, **i32),
                lengths=torch.tensor(length, **i32), ok=torch.tensor(oks), k=pools["k"], v=pools["v"])


def _exact_compact(case, s):
    table, n, free, shared = (s[k].tolist() for k in ("table", "n_blocks", "free", "shared"))
    unused = set(free[:int(s["n_free"])])
    used = {x for row, k in zip(table, n) for x in row[:k]}
    places = sorted(used | unused)
    front = places[:len(used)]
    moves = dict(zip(sorted(used - set(front)), sorted(set(front) - used)))
    pools = {}
    for name in ("k", "v"):
        pools[name] = s[name + "_pool"].double()
        pools[name][:, list(moves.values())] = pools[name][:, list(moves.keys())]
    new_shared = list(shared)
    for a, z in moves.items():
        new_shared[z], new_shared[a] = shared[a], 0
    back = places[len(used):][::-1]
    free[:len(back)] = back
    i32 = dict(dtype=torch.int32)
    return dict(table=torch.tensor([[moves.get(x, x) for x in row] for row in table], **i32), free=torch.tensor(free, **i32),
                n_free=torch.tensor([len(back)], **i32), shared=torch.tensor(new_shared, **i32),
                new_id=torch.tensor([moves.get(x, x) for x in range(len(shared))], **i32),
                n_used=torch.tensor([len(used)], **i32), k=pools["k"], v=pools["v"])


def _exact_chunk(case, s):
    ctx, n = s["sizes"]
    H, Hk, D, bs = case["H"], case["H_kv"], case["D"], case["bs"]
    if 4 * H * D * sum(k * (c + k) for c, k in zip(ctx, n)) > 5e12:
        return None
    outs, lses, at = [], [], 0
    for b, (c, k) in enumerate(zip(ctx, n)):
        rows = torch.arange(c + k, device=DEV)
        block = s["table"][b].long()[rows // bs]
        sees = rows[None, :] <= c + torch.arange(k, device=DEV)[:, None]
        o, z = [], []
        for h in range(H):
            kh, vh = (s[p][block, h // (H // Hk), rows % bs].double() for p in ("k_pool", "v_pool"))
            sc = s["q"][at:at + k, h].double() @ kh.T.contiguous() / math.sqrt(D)
            sc = sc.masked_fill(~sees, -math.inf)
            z.append(torch.logsumexp(sc, 1))
            o.append(torch.softmax(sc, 1) @ vh)
        at += k
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(z, 1))
    return dict(out=torch.cat(outs), lse=torch.cat(lses)) if case["lse"] else dict(out=torch.cat(outs))
