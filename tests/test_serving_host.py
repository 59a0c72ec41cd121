"""Refusals and host side of the operators around the block pool, without a
GPU: the library is a stand-in that records its arguments and must not be
reached by a call that is refused."""
from __future__ import annotations

import contextlib

import pytest
import torch

from test_block_pool_host import _pool, entries  # noqa: F401

I32, I64 = torch.int32, torch.int64


class _Lib:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.endswith("_workspace_size"):
            return lambda *a: 64

        def call(*a):
            self.calls.append((name, a))
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    from halo_amd import block_pool, rotate, tree, verify
    lib = _Lib()
    monkeypatch.setattr(block_pool.nat, "lib", lambda: lib)
    monkeypatch.setattr(block_pool.nat, "stream_ptr", lambda s=None: 0)
    for m in (block_pool, tree, rotate, verify):
        monkeypatch.setattr(m, "on_stream", lambda dev, stream: contextlib.nullcontext())
    return lib


def _i(*v, dtype=I32):
    return torch.tensor(v, dtype=dtype)


def _verify(**kw):
    d = dict(tokens=torch.zeros(5, dtype=I64), parents=torch.zeros(5, dtype=I32), cu_nodes=_i(0, 3, 5), probs=torch.ones(5, 7),
             accept=torch.zeros(5), sample=torch.zeros(2), max_nodes=3, draft_probs=torch.ones(5, 7))
    return {**d, **kw}


def _rotate(**kw):
    d = dict(q=torch.zeros(5, 4, 64), k=torch.zeros(5, 2, 64), v=torch.zeros(5, 2, 64), positions=torch.arange(5),
             cos=torch.ones(9, 32), sin=torch.ones(9, 32), slots=torch.arange(5), k_pool=torch.zeros(3, 2, 16, 64),
             v_pool=torch.zeros(3, 2, 16, 64), q_norm=torch.ones(64), k_norm=torch.ones(64))
    return {**d, **kw}


def _fork(**kw):
    d = dict(block_table=torch.zeros(2, 4, dtype=I32), n_blocks=_i(1, 1), free_blocks=torch.arange(9, dtype=I32), n_free=_i(9),
             shared=torch.zeros(12, dtype=I32), lengths=_i(5, 5), source=_i(0, 0), k_pool=torch.zeros(2, 12, 2, 16, 64),
             v_pool=torch.zeros(2, 12, 2, 16, 64))
    return {**d, **kw}


def _compact(**kw):
    d = _fork()
    d.pop("lengths")
    d.pop("source")
    return {**d, **kw}


def _chunk(**kw):
    d = dict(q=torch.zeros(5, 4, 64), k_pool=torch.zeros(3, 2, 16, 64), v_pool=torch.zeros(3, 2, 16, 64),
             block_table=torch.zeros(1, 3, dtype=I32), lengths=_i(1), cu_rows=_i(0, 5), max_rows=5)
    return {**d, **kw}


CALLS = dict(verify_tree=_verify, rotate_rows=_rotate, fork_blocks=_fork, compact_blocks=_compact, chunk_attention=_chunk)
_same = torch.zeros(3, 2, 16, 64)
_big = torch.zeros(2, 12, 2, 16, 64)
_flat = torch.zeros(64, dtype=I32)
_q = torch.zeros(5, 4, 64)

REFUSED = [
    ("verify_tree", dict(tokens=torch.zeros(5, dtype=I32))),
    ("verify_tree", dict(tokens=torch.zeros(4, dtype=I64))),
    ("verify_tree", dict(parents=torch.zeros(5, dtype=I64))),
    ("verify_tree", dict(parents=torch.zeros(10, dtype=I32)[::2])),
    ("verify_tree", dict(cu_nodes=_i(0))),
    ("verify_tree", dict(cu_nodes=_i(0, 3, 5, dtype=I64))),
    ("verify_tree", dict(probs=torch.ones(5, 7, dtype=torch.float64))),
    ("verify_tree", dict(probs=torch.ones(4, 7))),
    ("verify_tree", dict(probs=torch.ones(5, 14)[:, ::2])),
    ("verify_tree", dict(probs=torch.ones(5, 0))),
    ("verify_tree", dict(probs=torch.ones(5))),
    ("verify_tree", dict(draft_probs=torch.ones(5, 8))),
    ("verify_tree", dict(draft_probs=torch.ones(5, 7).half())),
    ("verify_tree", dict(draft_probs=torch.ones(7, 5).T)),
    ("verify_tree", dict(accept=torch.zeros(5, dtype=torch.float64))),
    ("verify_tree", dict(accept=torch.zeros(2))),
    ("verify_tree", dict(sample=torch.zeros(5))),
    ("verify_tree", dict(max_nodes=0)),
    ("verify_tree", dict(max_nodes=513)),
    ("verify_tree", dict(max_path=0)),
    ("verify_tree", dict(max_path=65)),
    ("rotate_rows", dict(q=torch.zeros(5, 4, 64).half())),
    ("rotate_rows", dict(q=torch.zeros(5, 256))),
    ("rotate_rows", dict(q=torch.zeros(4, 4, 64))),
    ("rotate_rows", dict(q=torch.zeros(5, 0, 64))),
    ("rotate_rows", dict(k=torch.zeros(5, 3, 64))),
    ("rotate_rows", dict(v=torch.zeros(5, 2, 64).bfloat16())),
    ("rotate_rows", dict(positions=torch.arange(4))),
    ("rotate_rows", dict(positions=torch.arange(5).float())),
    ("rotate_rows", dict(positions=torch.arange(10)[::2])),
    ("rotate_rows", dict(cos=torch.ones(9, 32).half(), sin=torch.ones(9, 32).half())),
    ("rotate_rows", dict(sin=torch.ones(8, 32))),
    ("rotate_rows", dict(cos=torch.ones(9, 40), sin=torch.ones(9, 40))),
    ("rotate_rows", dict(cos=torch.ones(9, 4), sin=torch.ones(9, 4))),
    ("rotate_rows", dict(cos=torch.ones(9, 12), sin=torch.ones(9, 12))),
    ("rotate_rows", dict(cos=torch.ones(0, 32), sin=torch.ones(0, 32))),
    ("rotate_rows", dict(cos=torch.ones(9, 64)[:, ::2], sin=torch.ones(9, 64)[:, ::2])),
    ("rotate_rows", dict(slots=torch.arange(5, dtype=I32))),
    ("rotate_rows", dict(q_norm=torch.ones(32))),
    ("rotate_rows", dict(k_norm=torch.ones(64).half())),
    ("rotate_rows", dict(k_norm=torch.ones(128)[::2])),
    ("rotate_rows", dict(eps=-1.0)),
    ("rotate_rows", dict(eps=float("inf"))),
    ("rotate_rows", dict(eps=float("nan"))),
    ("rotate_rows", dict(k_pool=_same, v_pool=_same)),
    ("rotate_rows", dict(k_pool=torch.zeros(1, 3, 2, 16, 64), v_pool=torch.zeros(1, 3, 2, 16, 64))),
    ("rotate_rows", dict(q=torch.zeros(5, 4, 96), k=torch.zeros(5, 2, 96), v=torch.zeros(5, 2, 96), q_norm=None, k_norm=None,
                         k_pool=torch.zeros(3, 2, 16, 96), v_pool=torch.zeros(3, 2, 16, 96))),
    ("rotate_rows", dict(k_pool=_same, v_pool=torch.zeros(3, 2, 16, 64), k=_same[1, :, :5].transpose(0, 1))),
    ("rotate_rows", dict(k_pool=_same, v_pool=torch.zeros(3, 2, 16, 64), q=_same.view(-1)[:1280].view(5, 4, 64))),
    ("rotate_rows", dict(k_pool=_same, v_pool=torch.zeros(3, 2, 16, 64), out=_same.view(-1)[:1280].view(5, 4, 64))),
    ("rotate_rows", dict(out=torch.zeros(5, 4, 64).half())),
    ("rotate_rows", dict(out=torch.zeros(5, 4, 32))),
    ("rotate_rows", dict(out=torch.zeros(1, 4, 64).expand(5, 4, 64))),
    ("rotate_rows", dict(q=_q, out=_q.as_strided((5, 4, 64), (64, 320, 1)))),
    ("fork_blocks", dict(block_table=torch.zeros(2, 4, dtype=I64))),
    ("fork_blocks", dict(block_table=torch.zeros(3, 4, dtype=I32))),
    ("fork_blocks", dict(n_blocks=_i(1))),
    ("fork_blocks", dict(n_free=_i(9, 9))),
    ("fork_blocks", dict(shared=torch.zeros(11, dtype=I32))),
    ("fork_blocks", dict(shared=torch.zeros(12, dtype=I64))),
    ("fork_blocks", dict(lengths=_i(5, 5, dtype=I64))),
    ("fork_blocks", dict(lengths=torch.zeros(0, dtype=I32))),
    ("fork_blocks", dict(source=_i(0))),
    ("fork_blocks", dict(source=_i(0, 0, dtype=I64))),
    ("fork_blocks", dict(n_blocks=_flat[:2], lengths=_flat[:2])),
    ("fork_blocks", dict(shared=_flat[:12], source=_flat[10:12])),
    ("fork_blocks", dict(shared=_flat[:12], free_blocks=_flat[11:20])),
    ("fork_blocks", dict(k_pool=_big, v_pool=_big)),
    ("fork_blocks", dict(k_pool=_big[:, :11], v_pool=torch.zeros(2, 11, 2, 16, 64))),
    ("fork_blocks", dict(v_pool=torch.zeros(2, 12, 2, 16, 64).half())),
    ("fork_blocks", dict(k_pool=torch.zeros(2, 1, 2, 16, 64).expand(2, 12, 2, 16, 64),
                         v_pool=torch.zeros(2, 1, 2, 16, 64).expand(2, 12, 2, 16, 64))),
    ("compact_blocks", dict(block_table=torch.zeros(2, 4))),
    ("compact_blocks", dict(n_blocks=torch.zeros(0, dtype=I32))),
    ("compact_blocks", dict(shared=torch.zeros(13, dtype=I32))),
    ("compact_blocks", dict(free_blocks=torch.zeros(18, dtype=I32)[::2])),
    ("compact_blocks", dict(n_blocks=_flat[:2], block_table=_flat[:8].view(2, 4))),
    ("compact_blocks", dict(k_pool=_big, v_pool=_big)),
    ("chunk_attention", dict(q=torch.zeros(5, 4, 1, 64))),
    ("chunk_attention", dict(q=torch.zeros(5, 4, 64).half())),
    ("chunk_attention", dict(q=torch.zeros(5, 3, 64))),
    ("chunk_attention", dict(max_rows=0)),
    ("chunk_attention", dict(cu_rows=_i(0, 2, 5))),
    ("chunk_attention", dict(lengths=_i(1, dtype=I64))),
    ("chunk_attention", dict(scale=0.0)),
    ("chunk_attention", dict(out=torch.zeros(5, 4, 32))),
    ("chunk_attention", dict(q=_q, out=_q)),
    ("chunk_attention", dict(lse=torch.zeros(4, 5))),
    ("chunk_attention", dict(out_dtype=torch.float64)),
]


@pytest.mark.parametrize("name,bad", REFUSED, ids=lambda x: x if isinstance(x, str) else "-".join(x))
def test_refused(lib, name, bad):
    import halo_amd
    with pytest.raises(AssertionError):
        getattr(halo_amd, name)(**CALLS[name](**bad))
    assert lib.calls == []


@pytest.mark.parametrize("name", CALLS)
def test_accepted_calls_reach_the_library(lib, name):
    import halo_amd
    getattr(halo_amd, name)(**CALLS[name]())
    assert [c[0] for c in lib.calls] == ["halo_" + ("chunk_attn" if name == "chunk_attention" else name)]


@pytest.mark.parametrize("name", CALLS)
def test_tensors_on_the_host_are_refused(monkeypatch, name):
    from halo_amd import block_pool
    import halo_amd
    lib = _Lib()
    monkeypatch.setattr(block_pool.nat, "lib", lambda: lib)
    with pytest.raises(AssertionError, match="GPU"):
        getattr(halo_amd, name)(**CALLS[name]())
    assert lib.calls == []


def test_rotate_in_place_and_row_forms(lib):
    """q, k and v of one projection; q in place; unaligned rows go through copies."""
    import halo_amd
    qkv = torch.zeros(5, 8, 64)
    d = _rotate(q=qkv[:, :4], k=qkv[:, 4:6], v=qkv[:, 6:])
    assert halo_amd.rotate_rows(**d, out=d["q"]) is d["q"]
    a = lib.calls[-1][1]
    assert a[1] == qkv.data_ptr() and a[2:4] == (512, 64) and a[11] == qkv.data_ptr()
    wide = torch.zeros(5, 8, 65)
    d = _rotate(q=wide[:, :4, 1:], k=wide[:, 4:6, 1:], v=wide[:, 6:, 1:])
    halo_amd.rotate_rows(**d)
    a = lib.calls[-1][1]
    assert a[2:4] == (256, 64) and a[6:8] == (128, 64)


# ---------------------------------------------------------------- the C entries' own checks

P = 4096


def _call(fn, d, kw):
    return fn(*{**d, **kw}.values())


def test_verify_entry_refuses(entries):  # noqa: F811
    d = dict(t=P, p=P, cu=P, B=2, N=5, mn=5, V=100, dt=0, pr=P, ps=100, q=P, qs=100, re=1, ac=P, sa=P, mp=4, pa=P, np=P, to=P,
             st=None)
    for kw in (dict(t=None), dict(cu=None), dict(pr=None), dict(sa=None), dict(to=None), dict(B=0), dict(B=70000), dict(N=-1),
               dict(mn=0), dict(mn=513), dict(V=0), dict(V=2 ** 24 + 1), dict(dt=5), dict(ps=-1), dict(qs=-1), dict(mp=0),
               dict(mp=65)):
        assert _call(entries.halo_verify_tree, d, kw) == -1, kw


def test_rotate_entry_refuses(entries):  # noqa: F811
    d = dict(pool=_pool(), q=P, qn=256, qh=64, H=4, k=P, kn=128, kh=64, v=P, vn=128, vh=64, o=P, on=256, oh=64, N=5, pos=P, p64=1,
             c=P, s=P, ts=32, tr=9, R=64, il=0, qw=P, qf=0, kw=P, kf=0, eps=1e-6, sl=P, st=None)
    for kw in (dict(pool=_pool(layers=2)), dict(pool=_pool(D=96)), dict(pool=_pool(k=4098)), dict(pool=_pool(sr=65)), dict(H=0),
               dict(N=-1), dict(R=0), dict(R=24), dict(R=80), dict(ts=31), dict(ts=34), dict(tr=0), dict(c=P + 4), dict(q=None),
               dict(q=P + 2), dict(qn=257), dict(kh=60), dict(vn=132), dict(o=P + 8), dict(oh=66), dict(pos=None), dict(sl=None),
               dict(eps=-1.0), dict(eps=float("nan")), dict(N=2 ** 29)):
        assert _call(entries.halo_rotate_rows, d, kw) == -1, kw


def test_fork_and_compact_entries_refuse(entries):  # noqa: F811
    d = dict(pool=_pool(), t=P, ts=4, n=P, B=2, W=4, f=P, cap=9, nf=P, sh=P, ln=P, src=P, new=2 * P, ok=P, ws=P,
             nb=entries.halo_fork_workspace_size(2, 4, 3), st=None)
    for kw in (dict(pool=_pool(dt=9)), dict(pool=_pool(blocks=0)), dict(t=None), dict(sh=None), dict(src=None), dict(ok=None),
               dict(B=0), dict(B=4097), dict(W=0), dict(ts=3), dict(cap=-1), dict(W=2 ** 30, ts=2 ** 30), dict(new=P), dict(ws=None),
               dict(ws=P + 4)):
        assert _call(entries.halo_fork_blocks, d, kw) == -1, kw
    assert _call(entries.halo_fork_blocks, d, dict(nb=d["nb"] - 1)) == -4
    d = dict(pool=_pool(), t=P, ts=4, n=P, B=2, W=4, f=P, cap=9, nf=P, sh=P, new=P, nu=P, ws=P,
             nb=entries.halo_compact_workspace_size(3), st=None)
    for kw in (dict(pool=_pool(dt=9)), dict(t=None), dict(sh=None), dict(new=None), dict(nu=None), dict(B=0), dict(W=0), dict(ts=3),
               dict(cap=-1), dict(W=2 ** 30, ts=2 ** 30), dict(ws=None), dict(ws=P + 4)):
        assert _call(entries.halo_compact_blocks, d, kw) == -1, kw
    assert _call(entries.halo_compact_blocks, d, dict(nb=d["nb"] - 1)) == -4


@pytest.mark.parametrize("N,rows", [(200, 5), (200, 600), (700, 5), (700, 600)])
def test_chunk_entry_refuses(entries, N, rows):  # noqa: F811
    need = entries.halo_chunk_workspace_size(1, 1, N, 4, 2, 64, 3 * 16, rows)
    d = dict(pool=_pool(), q=P, qn=256, qh=64, N=N, H=4, table=P, ts=3, B=1, W=3, ln=P, cu=P, mr=rows, scale=0.125, out=P, on=256,
             oh=64, odt=1, lse=None, ws=P, nb=max(need, 1 << 20), st=None)
    for kw in (dict(pool=_pool(dt=3)), dict(pool=_pool(D=96)), dict(pool=_pool(layers=2)), dict(pool=_pool(k=4104)), dict(H=5),
               dict(H=0), dict(B=0), dict(W=0), dict(mr=0), dict(q=4100), dict(q=None), dict(qn=257), dict(table=None), dict(ts=2),
               dict(scale=0.0), dict(out=None), dict(odt=7), dict(out=4100), dict(N=-1)):
        assert _call(entries.halo_chunk_attn, d, kw) == -1, kw
    if N > 256:
        for kw in (dict(B=4097), dict(N=2 ** 30), dict(W=2 ** 27 - 128, ts=2 ** 27, N=2000), dict(ws=None), dict(ws=P + 4)):
            assert _call(entries.halo_chunk_attn, d, kw) == -1, kw
        assert need > 0 and _call(entries.halo_chunk_attn, d, dict(nb=need - 1)) == -4
