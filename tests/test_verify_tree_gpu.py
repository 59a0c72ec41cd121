"""Verification of drafted trees on the GPU.

Tokens and paths are whole numbers and equal the definition in float64: a draw
falls between two sums of float64 terms in another order with a chance of about
1e-13 a token."""
from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle import serving

pytestmark = pytest.mark.gpu
DT = [torch.float32, torch.bfloat16, torch.float16]


class Case:
    def __init__(self, dev, *, nodes, V, fan=3, draft="with", dtype=torch.float32, seed=0, max_path=None, pad=0, spread=2.0,
                 noise=0.7, stride=0):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.cu = np.concatenate([[0], np.cumsum(nodes)]).tolist()
        N = self.cu[-1] + pad
        logits = torch.randn(N, V, generator=g) * spread
        self.probs = torch.softmax(logits, 1).to(dtype)
        q = torch.softmax(logits + noise * torch.randn(N, V, generator=g), 1).to(dtype)
        self.parents, self.tokens = [], []
        for b, n in enumerate(nodes):
            parents, count = [-1], [0]
            for i in range(1, n):
                free = [p for p in range(i) if count[p] < fan]
                p = rng.choice(free[:4])
                parents.append(p)
                count[p] += 1
                count.append(0)
            kids = {}
            for i in range(n):
                p = parents[i]
                if p < 0:
                    self.tokens.append(rng.randrange(V))
                    continue
                row = q[self.cu[b] + p].double()
                if p not in kids:
                    if draft == "none":
                        kids[p] = row.argsort(descending=True, stable=True)[:fan].tolist() * fan
                    else:
                        m = min(fan, int((row > 0).sum())) if draft == "without" else fan
                        kids[p] = torch.multinomial(row, m, replacement=draft == "with", generator=g).tolist() + [-1] * fan
                self.tokens.append(kids[p].pop(0))
            self.parents += parents[:n]
        self.tokens += [0] * pad
        self.parents += [0] * pad
        self.draft = None if draft == "none" else q
        self.replacement = draft != "without"
        self.accept = torch.rand(N, generator=g)
        self.sample = torch.rand(len(nodes), generator=g)
        self.max_nodes, self.V, self.stride = max(max(nodes), 1), V, stride
        self.max_path = max_path or min(self.max_nodes, 64)
        self.dev = dev

    def args(self):
        d = self.dev

        def rows(t):
            if t is None or not self.stride:
                return t if t is None else t.to(d)
            wide = torch.full((t.shape[0], t.shape[1] + self.stride), 9.0, dtype=t.dtype, device=d)
            wide[:, 1:1 + t.shape[1]] = t.to(d)
            return wide[:, 1:1 + t.shape[1]]
        return dict(tokens=torch.tensor(self.tokens, dtype=torch.int64, device=d),
                    parents=torch.tensor(self.parents, dtype=torch.int32, device=d),
                    cu_nodes=torch.tensor(self.cu, dtype=torch.int32, device=d), probs=rows(self.probs),
                    accept=self.accept.to(d), sample=self.sample.to(d), max_nodes=self.max_nodes,
                    draft_probs=rows(self.draft), replacement=self.replacement, max_path=self.max_path)

    def exact(self):
        return serving.verify(self.tokens, self.parents, self.cu, self.probs.double().numpy(), self.accept.double().tolist(),
                              self.sample.double().tolist(), max_nodes=self.max_nodes,
                              draft=None if self.draft is None else self.draft.double().numpy(),
                              replacement=self.replacement, max_path=self.max_path)

    def check(self, got=None, **kw):
        import halo_amd
        got = got or halo_amd.verify_tree(**{**self.args(), **kw})
        path, n_path, token = self.exact()
        assert got.path.dtype == got.n_path.dtype == torch.int32 and got.token.dtype == torch.int64
        assert got.n_path.tolist() == n_path
        assert got.path.tolist() == path
        assert got.token.tolist() == token
        return n_path


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("draft", ["none", "with", "without"])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 2048, 2049, 5003])
def test_vocabularies(dev, V, draft, dtype):
    Case(dev, nodes=[9, 1, 5, 12, 3, 7], V=V, fan=min(3, V), draft=draft, dtype=dtype, seed=V).check()


@pytest.mark.parametrize("draft", ["none", "with", "without"])
@pytest.mark.parametrize("V", [50001, 131072])
def test_large_vocabularies(dev, V, draft):
    Case(dev, nodes=[6, 9], V=V, draft=draft, seed=V, spread=3.0).check()


@pytest.mark.parametrize("draft", ["none", "with", "without"])
@pytest.mark.parametrize("noise", [0.1, 3.0])
@pytest.mark.parametrize("fan", [1, 8])
def test_many_accepted_and_many_rejected(dev, fan, noise, draft):
    n = Case(dev, nodes=[40] * 20, V=300, fan=fan, draft=draft, seed=fan, noise=noise).check()
    assert max(n) >= 2 if noise < 1 else min(n) == 1


@pytest.mark.parametrize("draft", ["none", "with", "without"])
def test_wide_nodes(dev, draft):
    """Up to 511 children of one node, most of them rejected."""
    c = Case(dev, nodes=[512, 70, 130, 256], V=900, fan=600, draft=draft, seed=4, noise=4.0, spread=0.3)
    for b in range(4):
        for i in range(c.cu[b] + 1, c.cu[b + 1]):
            c.parents[i] = 0
    g = torch.Generator().manual_seed(1)
    for b in range(4):
        n = c.cu[b + 1] - c.cu[b]
        row = torch.ones(900, dtype=torch.float64) if c.draft is None else c.draft[c.cu[b]].double()
        c.tokens[c.cu[b] + 1:c.cu[b + 1]] = torch.multinomial(row, n - 1, replacement=draft == "with", generator=g).tolist()
    c.accept = 1 - (1 - c.accept) * 1e-3
    c.check()


@pytest.mark.parametrize("draft", ["none", "with", "without"])
def test_depths(dev, draft):
    for max_path in (1, 2, 5, 64):
        c = Case(dev, nodes=[90, 70, 2, 1], V=40, fan=1, draft=draft, seed=max_path, noise=0.01, max_path=max_path)
        c.accept *= 0.05
        n = c.check()
        assert max(n) == max_path


def test_default_path_length(dev):
    import halo_amd
    c = Case(dev, nodes=[5, 3], V=11)
    a = c.args()
    a.pop("max_path")
    assert halo_amd.verify_tree(**a).path.shape == (2, 5)


@pytest.mark.parametrize("draft", ["none", "with", "without"])
def test_empty_padded_and_cut_requests(dev, draft):
    c = Case(dev, nodes=[0, 7, 0, 12, 1, 0], V=77, draft=draft, seed=3, pad=5)
    c.check()
    c.max_nodes = 6  # nodes 6 .. of a request are left out
    c.check()
    c.max_nodes = 12
    for cu in ([0, 7, 7, 4, 30, 30, 99], [-7, 2 ** 30, -2 ** 31, 2 ** 31 - 1, 0, 19, -1]):  # falling, and past the nodes
        c.cu = cu
        c.check()


@pytest.mark.parametrize("draft", ["none", "with", "without"])
def test_odd_nodes(dev, draft):
    """Tokens outside the vocabulary, further roots, parents that are no earlier node, the same token twice."""
    c = Case(dev, nodes=[12, 14, 9, 30], V=50, fan=6, draft=draft, seed=9, noise=2.0)
    c.tokens[3] = -1
    c.tokens[5] = 50
    c.tokens[13] = 2 ** 40
    for b, i, p in ((0, 4, -7), (1, 6, 6), (1, 8, 13), (2, 3, -1), (3, 9, 2 ** 30)):
        c.parents[c.cu[b] + i] = p
    lo = c.cu[3]
    for i in range(1, 12):
        c.parents[lo + i] = 0
        c.tokens[lo + i] = [3, 3, 8, 3, 8, 11, 11, 3, 20, 21, 22][i - 1]
    c.accept[lo + 1:lo + 12] = 0.999
    c.check()


@pytest.mark.parametrize("draft", ["none", "with", "without"])
@pytest.mark.parametrize("u", [0.0, 1 - 2.0 ** -24])
def test_ends_of_the_random_numbers(dev, u, draft):
    c = Case(dev, nodes=[6, 1, 9, 4], V=333, draft=draft, seed=1)
    c.probs[:, ::3] = 0
    c.probs[:, -5:] = 0
    c.sample.fill_(u)
    c.check()
    c.accept.fill_(u)
    c.check()


@pytest.mark.parametrize("draft", ["none", "with", "without"])
def test_nothing_left(dev, draft):
    """Target and draft agree on tokens that are rejected all the same: q = p, and p in one token."""
    c = Case(dev, nodes=[5, 5, 5], V=64, fan=4, draft=draft, seed=2)
    if c.draft is not None:
        c.draft.copy_(c.probs)
    c.probs[5:10] = 0
    c.probs[5:10, 7] = 1.0
    if c.draft is not None:
        c.draft[5:10] = c.probs[5:10]
    c.tokens[6:10] = [7, 7, 7, 7]
    c.accept.fill_(float("nan"))  # nothing is accepted
    c.check()


def test_nan_negative_and_zero_probabilities(dev):
    for draft in ("none", "with", "without"):
        c = Case(dev, nodes=[8, 8, 8], V=100, draft=draft, seed=5)
        c.probs[0, 3:9] = float("nan")
        c.probs[1, ::2] = -0.5
        c.probs[2] = 0
        if c.draft is not None:
            c.draft[0, 5:20] = float("nan")
            c.draft[1, ::3] = -1
        c.probs[16:24] = 0
        c.check()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("stride", [1, 5, 64])
def test_row_strides(dev, stride, dtype):
    """Rows that begin at any element; the places between them hold 9."""
    Case(dev, nodes=[9, 4], V=4099, dtype=dtype, seed=stride, stride=stride).check()
    Case(dev, nodes=[9, 4], V=130, dtype=dtype, seed=stride, stride=stride, draft="none").check()


def test_one_row_for_all_nodes(dev):
    import halo_amd
    c = Case(dev, nodes=[6, 5], V=200, seed=8)
    c.probs = c.probs[:1].expand(11, 200)
    c.draft = c.draft[:1].expand(11, 200)
    a = c.args()
    a["probs"], a["draft_probs"] = c.probs[:1].to(dev).expand(11, 200), c.draft[:1].to(dev).expand(11, 200)
    c.check(halo_amd.verify_tree(**a))


@pytest.mark.parametrize("B", [300, 1500])
def test_many_requests(dev, B):
    rng = random.Random(B)
    Case(dev, nodes=[rng.randint(0, 6) for _ in range(B)], V=61, seed=B).check()


def test_rows_past_32_bit_offsets(dev):
    """Row numbers times the row length beyond 2^32 elements."""
    import halo_amd
    N, V = 33000, 131072
    probs = torch.zeros((N, V), device=dev, dtype=torch.bfloat16)
    lo = N - 3
    probs[lo, 5], probs[lo + 1, 100000], probs[lo + 2, 99] = 1, 1, 1
    z = dict(device=dev, dtype=torch.int32)
    tokens = torch.zeros(N, device=dev, dtype=torch.int64)
    tokens[lo + 1], tokens[lo + 2] = 5, 100000
    parents = torch.zeros(N, **z)
    parents[lo + 1], parents[lo + 2] = 0, 1
    got = halo_amd.verify_tree(tokens, parents, torch.tensor([lo, N], **z), probs, torch.full((N,), 0.5, device=dev),
                               torch.full((1,), 0.5, device=dev), max_nodes=3)
    assert got.path.tolist() == [[0, 1, 2]] and got.token.tolist() == [99]


@pytest.mark.parametrize("draft", ["none", "with", "without"])
def test_tokens_have_the_targets_distribution(dev, draft):
    """Two-step trees: the first new token of 60 000 requests against p; each share within 5 standard deviations."""
    import halo_amd
    B, V, fan = 60000, 6, 3
    g = torch.Generator(device=dev).manual_seed(0)
    p = torch.tensor([0.35, 0.05, 0.2, 0.1, 0.0, 0.3], device=dev)
    q = torch.tensor([0.1, 0.3, 0.15, 0.05, 0.2, 0.2], device=dev)
    n = 1 + fan
    if draft == "none":
        kids = torch.tensor([[1, 4, 2]], device=dev).expand(B, fan)
    else:
        kids = torch.multinomial(q.expand(B, V), fan, replacement=draft == "with", generator=g)
    tokens = torch.cat([torch.zeros(B, 1, dtype=torch.int64, device=dev), kids], 1).reshape(-1)
    parents = torch.tensor([-1, 0, 0, 0], device=dev, dtype=torch.int32).repeat(B)
    got = halo_amd.verify_tree(tokens, parents, torch.arange(B + 1, device=dev, dtype=torch.int32) * n, p.expand(B * n, V),
                               torch.rand(B * n, generator=g, device=dev), torch.rand(B, generator=g, device=dev), max_nodes=n,
                               draft_probs=None if draft == "none" else q.expand(B * n, V), replacement=draft != "without")
    second = got.path[:, 1].long()
    first = torch.where(second > 0, tokens.view(B, n).gather(1, second.clamp(min=0)[:, None])[:, 0], got.token)
    share = torch.bincount(first, minlength=V).double() / B
    sd = (p.double() * (1 - p.double()) / B).sqrt()
    assert bool(((share - p.double()).abs() <= 5 * sd).all())
    assert 0.2 < (second > 0).double().mean().item() < 0.95


def test_replayed_on_another_stream_and_side_by_side(dev):
    import halo_amd
    cases = [Case(dev, nodes=[9, 3, 12], V=5000, seed=i, draft=d) for i, d in enumerate(("with", "none"))]
    a = cases[0].args()
    other = Case(dev, nodes=[9, 3, 12], V=5000, seed=7)
    b = other.args()
    halo_amd.verify_tree(**a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = halo_amd.verify_tree(**a)
    for turn in range(4):
        src = (a, cases[0]) if turn % 2 == 0 else (b, other)
        if turn == 1:
            for k in ("tokens", "parents", "probs", "draft_probs", "accept", "sample"):
                a[k].copy_(b[k])
        if turn == 2:
            first = cases[0].args()
            for k in ("tokens", "parents", "probs", "draft_probs", "accept", "sample"):
                a[k].copy_(first[k])
        if turn == 3:
            for k in ("tokens", "parents", "probs", "draft_probs", "accept", "sample"):
                a[k].copy_(b[k])
        graph.replay()
        src[1].check(got)
        cases[1].check()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    args = [c.args() for c in cases]
    torch.cuda.synchronize()
    got = [halo_amd.verify_tree(**x, stream=s) for x, s in zip(args, (s1, s2))]
    torch.cuda.synchronize()
    for c, r in zip(cases, got):
        c.check(r)


@pytest.mark.parametrize("draft", ["none", "with", "without"])
@pytest.mark.parametrize("V", [131073, 151936, 2 ** 20 + 77])
def test_vocabularies_of_several_narrowing_rounds(dev, V, draft):
    """More than 131072 tokens: the range that holds the last token is found in two rounds and more, each with the rejected
    tokens left out."""
    c = Case(dev, nodes=[5, 3], V=V, draft=draft, seed=V, spread=3.0)
    c.check()
    c.accept = 1 - c.accept * 2.0 ** -10  # most children are rejected
    for u in (0.0, 0.25, 0.999, 1 - 2.0 ** -24):
        c.sample.fill_(u)
        c.check()
    c.probs[:, :-40] = 0  # everything in the last range
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        c.sample.fill_(u)
        c.check()


@pytest.mark.parametrize("draft", ["none", "with", "without"])
def test_a_vocabulary_near_the_largest(dev, draft):
    c = Case(dev, nodes=[2], V=2 ** 24 - 5, draft=draft, dtype=torch.bfloat16, seed=1, fan=1)
    for u in (0.0, 0.7, 1 - 2.0 ** -24):
        c.sample.fill_(u)
        c.check()
    c.accept.fill_(1 - 2.0 ** -24)
    c.probs[:, :2 ** 23] = 0
    c.check()


@pytest.mark.parametrize("dtype", DT)
def test_rejected_tokens_whose_marks_are_the_same(dev, dtype):
    """Without draft probabilities rejected tokens are found by marks that tokens 131072 apart share."""
    V, far = 3 * 131072 + 11, 131072
    kids = [40, 40 + far, 41, 47 + 2 * far, 3 * far + 3, 9 + far, V - 1, 40, far - 1]
    c = Case(dev, nodes=[1 + len(kids)] * 4, V=V, draft="none", dtype=dtype, seed=6)
    c.probs[:] = 0
    near = sorted({min(max(t + d, 0), V - 1) for t in kids for d in range(-9, 10)} | {t % far for t in kids} | {t % far + far for t in kids})
    g = torch.Generator().manual_seed(7)
    for b in range(4):
        lo = c.cu[b]
        c.probs[lo:lo + 10, near] = (torch.rand(10, len(near), generator=g) / len(near)).to(dtype)
        c.parents[lo + 1:lo + 10], c.tokens[lo + 1:lo + 10] = [0] * 9, kids
    c.accept.fill_(1 - 2.0 ** -24)
    for u in (0.0, 0.1, 0.35, 0.6, 0.85, 1 - 2.0 ** -24):
        c.sample = torch.tensor([u, u * 0.99, u * 0.9, u * 0.7])
        assert c.check() == [1] * 4


@pytest.mark.parametrize("draft", ["none", "with", "without"])
@pytest.mark.parametrize("share", [0.25, 0.9, 1.5])
def test_rows_that_do_not_sum_to_one(dev, draft, share):
    """Z begins at 1 whatever p sums to; without draft probabilities it is 1 less the rejected tokens' p, not the sum of what
    is left."""
    c = Case(dev, nodes=[12, 30, 7, 25], V=90, fan=5, draft=draft, seed=12, noise=1.5)
    c.probs *= share
    c.check()
