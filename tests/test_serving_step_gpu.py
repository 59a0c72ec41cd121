"""The operators of a serving step together: prompts admitted, rotated, written
and attended, samples forked from them, trees drafted, attended, verified and
committed, requests given up and the pool compacted; against the same attention
over each request's rows kept apart."""
from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu
I32 = torch.int32


class Model:
    """One attention layer: q, k and v of a token are a table's rows, rotated by position and normed."""

    def __init__(self, dev, V=50, H=4, Hk=2, D=64, dtype=torch.float32):
        g = torch.Generator().manual_seed(0)
        self.qkv = torch.randn(V, H + 2 * Hk, D, generator=g).to(dtype).to(dev)
        self.head = torch.randn(H * D, V, generator=g).to(dev) * 0.2
        angle = torch.arange(2000, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, D, 2).double() / D)
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        self.w = (1 + 0.1 * torch.randn(D, generator=g)).to(dtype).to(dev)
        self.H, self.Hk, self.D, self.dev = H, Hk, D, dev

    def plain(self, tokens, positions, sees):
        """float64: outputs of these tokens at these positions, row i attending the rows of ``sees[i]``."""
        x = self.qkv[tokens].double()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * self.w.double()
        c, s = (t.double()[positions][:, None] for t in (self.cos, self.sin))
        a, b = y[..., :self.D // 2], y[..., self.D // 2:]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
        q, k, v = y[:, :self.H], y[:, self.H:self.H + self.Hk], x[:, self.H + self.Hk:]
        rep = self.H // self.Hk
        k, v = (t.repeat_interleave(rep, 1).transpose(0, 1).contiguous() for t in (k, v))
        sc = torch.stack([qh @ kh.T.contiguous() for qh, kh in zip(q.transpose(0, 1), k)]) * self.D ** -0.5
        p = torch.softmax(sc.masked_fill(~sees, -torch.inf), -1)
        return torch.stack([ph @ vh for ph, vh in zip(p, v)], 1)


def test_a_run_of_steps(dev):
    import halo_amd
    m = Model(dev)
    rng = random.Random(1)
    g = torch.Generator(device=dev).manual_seed(2)
    B, bs, P, W, V, n = 6, 16, 400, 80, 50, 7
    kp, vp = (torch.zeros(1, P, m.Hk, bs, m.D, device=dev) for _ in range(2))
    table = torch.full((B, W), -1, dtype=I32, device=dev)
    owned, lengths = torch.zeros(B, dtype=I32, device=dev), torch.zeros(B, dtype=I32, device=dev)
    free, n_free = torch.randperm(P, generator=g, device=dev).to(I32), torch.tensor([P], dtype=I32, device=dev)
    shared = torch.zeros(P, dtype=I32, device=dev)
    text = [[] for _ in range(B)]  # each request's tokens

    def write(tokens, positions, up):
        x = m.qkv[tokens]
        return halo_amd.rotate_rows(x[:, :m.H], x[:, m.H:m.H + m.Hk], x[:, m.H + m.Hk:], positions, m.cos, m.sin, up.slots, kp[0],
                                    vp[0], q_norm=m.w, k_norm=m.w)

    def near(got, want):
        assert float((got.double() - want).abs().max()) < 2e-5

    # prompts of requests 0 and 3, one of them longer than the tree kernels take
    new = [700, 0, 0, 33, 0, 0]
    for b in range(B):
        text[b] = [rng.randrange(V) for _ in range(new[b])]
    up = halo_amd.update_block_tables(table, owned, free, n_free, torch.tensor(new, dtype=I32, device=dev), lengths, block_size=bs,
                                      max_rows=sum(new))
    tokens = torch.tensor(text[0] + text[3], device=dev)
    positions = torch.cat([torch.arange(700, device=dev), torch.arange(33, device=dev)])
    q = write(tokens, positions, up)
    out = halo_amd.chunk_attention(q, kp[0], vp[0], table, lengths, up.cu_rows, max_rows=700)
    causal = torch.ones(700, 700, dtype=torch.bool, device=dev).tril()
    near(out[:700], m.plain(tokens[:700], positions[:700], causal))
    near(out[700:], m.plain(tokens[700:], positions[700:], causal[:33, :33]))
    lengths = torch.tensor(new, dtype=I32, device=dev)
    # samples of both
    lengths, ok = halo_amd.fork_blocks(table, owned, free, n_free, shared, lengths,
                                       torch.tensor([0, 0, 0, 3, 3, -1], dtype=I32, device=dev), kp, vp)
    assert ok.item() and lengths.tolist() == [700, 700, 700, 33, 33, 0]
    text = [list(text[a]) if a >= 0 else [] for a in (0, 0, 0, 3, 3, -1)]
    last = [rng.randrange(V) for _ in range(B)]  # sampled behind the prompts
    for step in range(6):
        live = [b for b in range(B) if text[b]]
        drafted = [n if b in live else 0 for b in range(B)]
        parents = [[-1, 0, 0, 1, 1, 2, 4] if b in live else [] for b in range(B)]
        flat = torch.tensor([p for x in parents for p in x], dtype=I32, device=dev)
        want_len = lengths + torch.tensor(drafted, dtype=I32, device=dev)
        up = halo_amd.update_block_tables(table, owned, free, n_free, want_len, lengths, block_size=bs, max_rows=B * n)
        assert up.ok.all()
        N = sum(drafted)
        mask, depth = halo_amd.tree_layout(flat, up.cu_rows, max_nodes=n)
        nodes = [[last[b]] + [rng.randrange(V) for _ in range(n - 1)] if b in live else [] for b in range(B)]
        tokens = torch.tensor([t for x in nodes for t in x], device=dev)
        owner = torch.tensor([b for b in range(B) for _ in range(drafted[b])], device=dev)
        positions = lengths[owner].long() + depth
        q = write(tokens, positions, halo_amd.BlockUpdate(up.cu_rows, up.slots[:N], up.ok))
        out = halo_amd.tree_attention(q, kp[0], vp[0], table, lengths, up.cu_rows, mask=mask, max_nodes=n)
        at = 0
        for b in live:  # every node sees its request's text and its own path
            c = len(text[b])
            rows = torch.tensor(text[b] + nodes[b], device=dev)
            sees = torch.ones(c + n, c + n, dtype=torch.bool, device=dev).tril()
            tree = torch.zeros(n, n, dtype=torch.bool, device=dev)
            for i in range(n):
                j = i
                while j >= 0:
                    tree[i, j] = True
                    j = parents[b][j]
            sees[c:, c:] = tree
            pos = torch.cat([torch.arange(c, device=dev), positions[at:at + n]])
            near(out[at:at + n], m.plain(rows, pos, sees)[c:])
            at += n
        probs = torch.softmax(out.reshape(N, -1) @ m.head, 1)
        got = halo_amd.verify_tree(tokens, flat, up.cu_rows, probs, torch.rand(N, generator=g, device=dev) * 0.05,
                                   torch.rand(B, generator=g, device=dev), max_nodes=n)
        lengths = halo_amd.commit_path(kp, vp, table, lengths, got.path, got.n_path)
        path, count, token = got.path.tolist(), got.n_path.tolist(), got.token.tolist()
        for b in range(B):
            assert (count[b] == 0) == (b not in live) and (token[b] == -1) == (b not in live)
            text[b] += [nodes[b][i] for i in path[b][:count[b]]]
            last[b] = token[b]
        assert lengths.tolist() == [len(t) for t in text]
        if step in (1, 3):
            source = [[1, 1, -1, 3, 4, 4], [0, 0, 1, 1, -1, 5]][step // 2]
            # room behind the committed rows goes back before rows are shared
            halo_amd.update_block_tables(table, owned, free, n_free, lengths, lengths, block_size=bs, max_rows=0)
            lengths, ok = halo_amd.fork_blocks(table, owned, free, n_free, shared, lengths,
                                               torch.tensor(source, dtype=I32, device=dev), kp, vp)
            assert ok.item()
            text = [list(text[a]) if a >= 0 else [] for a in source]
            last = [last[a] if a >= 0 else 0 for a in source]
            new_id, used = halo_amd.compact_blocks(table, owned, free, n_free, shared, kp, vp)
            held = {x for row, k in zip(table.tolist(), owned.tolist()) for x in row[:k]}
            assert held == set(range(used.item())) and n_free.item() == P - used.item()
    assert max(len(t) for t in text) > 706
    lengths, ok = halo_amd.fork_blocks(table, owned, free, n_free, shared, lengths, torch.full((B,), -1, dtype=I32, device=dev), kp, vp)
    assert sorted(free.tolist()) == list(range(P)) and n_free.item() == P and not shared.any()
