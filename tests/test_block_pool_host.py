"""Refusals and host side of the block-pool operators, without a GPU: the
library is a stand-in that records its arguments and must not be reached by a
call that is refused."""
from __future__ import annotations

import contextlib
import ctypes
import struct

import pytest
import torch

I32, I64 = torch.int32, torch.int64


class _Lib:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name == "halo_tree_workspace_size":
            return lambda *a: 0

        def call(*a):
            self.calls.append((name, a))
            return 0
        return call


@pytest.fixture
def lib(monkeypatch):
    from halo_amd import block_pool, tree
    lib = _Lib()
    monkeypatch.setattr(block_pool.nat, "lib", lambda: lib)
    monkeypatch.setattr(block_pool.nat, "stream_ptr", lambda s=None: 0)
    for m in (block_pool, tree):
        monkeypatch.setattr(m, "on_stream", lambda dev, stream: contextlib.nullcontext())
    return lib


def _tables(**kw):
    d = dict(block_table=torch.zeros(2, 4, dtype=I32), n_blocks=torch.zeros(2, dtype=I32),
             free_blocks=torch.arange(9, dtype=I32), n_free=torch.full((1,), 9, dtype=I32),
             lengths=torch.ones(2, dtype=I32), first=torch.zeros(2, dtype=I32), block_size=16, max_rows=4)
    return {**d, **kw}


def _append(**kw):
    d = dict(k_new=torch.zeros(5, 2, 64), v_new=torch.zeros(5, 2, 64), slots=torch.arange(5),
             k_pool=torch.zeros(3, 2, 16, 64), v_pool=torch.zeros(3, 2, 16, 64))
    return {**d, **kw}


def _layout(**kw):
    return {**dict(parents=torch.zeros(5, dtype=I32), cu_nodes=torch.tensor([0, 5], dtype=I32), max_nodes=5), **kw}


def _attend(**kw):
    d = dict(q=torch.zeros(5, 4, 64), k_pool=torch.zeros(3, 2, 16, 64), v_pool=torch.zeros(3, 2, 16, 64),
             block_table=torch.zeros(1, 3, dtype=I32), lengths=torch.ones(1, dtype=I32),
             cu_nodes=torch.tensor([0, 5], dtype=I32), max_nodes=5, mask=torch.zeros(5, 1, dtype=I64))
    return {**d, **kw}


def _commit(**kw):
    d = dict(k_pool=torch.zeros(2, 3, 2, 16, 64), v_pool=torch.zeros(2, 3, 2, 16, 64),
             block_table=torch.zeros(2, 3, dtype=I32), lengths=torch.ones(2, dtype=I32),
             path=torch.zeros(2, 4, dtype=I32), n_path=torch.ones(2, dtype=I32))
    return {**d, **kw}


CALLS = dict(update_block_tables=_tables, append_rows=_append, tree_layout=_layout, tree_attention=_attend,
             commit_path=_commit)
_same = torch.zeros(3, 2, 16, 64)
_lengths = torch.ones(2, dtype=I32)
_q = torch.zeros(5, 4, 64)
_out = torch.zeros(5, 4, 64)
_path = torch.zeros(2, 1, dtype=I32)

REFUSED = [
    ("update_block_tables", dict(block_table=torch.zeros(2, 4, dtype=I64))),
    ("update_block_tables", dict(block_table=torch.zeros(3, 4, dtype=I32))),
    ("update_block_tables", dict(block_table=torch.zeros(4, 2, dtype=I32).T)),
    ("update_block_tables", dict(block_table=torch.zeros(1, 4, dtype=I32).expand(2, 4))),
    ("update_block_tables", dict(block_table=torch.zeros(2, 0, dtype=I32))),
    ("update_block_tables", dict(n_blocks=torch.zeros(3, dtype=I32))),
    ("update_block_tables", dict(n_blocks=_lengths, lengths=_lengths)),
    ("update_block_tables", dict(n_free=torch.zeros((), dtype=I32))),
    ("update_block_tables", dict(free_blocks=torch.zeros(18, dtype=I32)[::2])),
    ("update_block_tables", dict(lengths=torch.ones(2))),
    ("update_block_tables", dict(first=torch.ones(1, dtype=I32))),
    ("update_block_tables", dict(block_size=0)),
    ("update_block_tables", dict(max_rows=-1)),
    ("update_block_tables", dict(lengths=torch.ones(0, dtype=I32))),
    ("append_rows", dict(k_new=torch.zeros(5, 2, 64).half())),
    ("append_rows", dict(k_new=torch.zeros(4, 2, 64))),
    ("append_rows", dict(v_new=torch.zeros(5, 3, 64))),
    ("append_rows", dict(v_new=torch.zeros(5, 2, 128)[..., ::2])),
    ("append_rows", dict(slots=torch.arange(5, dtype=I32))),
    ("append_rows", dict(v_pool=torch.zeros(3, 2, 16, 64).half())),
    ("append_rows", dict(v_pool=torch.zeros(3, 2, 8, 64))),
    ("append_rows", dict(v_pool=torch.zeros(3, 16, 2, 64).transpose(1, 2))),
    ("append_rows", dict(k_pool=_same, v_pool=_same)),
    ("append_rows", dict(k_pool=torch.zeros(1, 2, 16, 64).expand(3, 2, 16, 64),
                         v_pool=torch.zeros(1, 2, 16, 64).expand(3, 2, 16, 64))),
    ("append_rows", dict(k_pool=torch.zeros(2, 3, 2, 16, 64), v_pool=torch.zeros(2, 3, 2, 16, 64))),
    ("append_rows", dict(k_pool=torch.zeros(3, 2, 16, 64, dtype=torch.float64),
                         v_pool=torch.zeros(3, 2, 16, 64, dtype=torch.float64))),
    ("append_rows", dict(k_pool=_same, v_pool=torch.zeros(3, 2, 16, 64), k_new=_same[1, :, :5].transpose(0, 1))),
    ("tree_layout", dict(max_nodes=0)),
    ("tree_layout", dict(max_nodes=513)),
    ("tree_layout", dict(parents=torch.zeros(5, dtype=I64))),
    ("tree_layout", dict(cu_nodes=torch.tensor([0], dtype=I32))),
    ("tree_layout", dict(mask=torch.zeros(5, 2, dtype=I64))),
    ("tree_layout", dict(depth=torch.zeros(5, dtype=I64))),
    ("tree_attention", dict(q=torch.zeros(5, 4, 1, 64))),
    ("tree_attention", dict(q=torch.zeros(5, 4, 64).half())),
    ("tree_attention", dict(q=torch.zeros(5, 3, 64))),
    ("tree_attention", dict(q=torch.zeros(5, 4, 96), k_pool=torch.zeros(3, 2, 16, 96), v_pool=torch.zeros(3, 2, 16, 96))),
    ("tree_attention", dict(k_pool=torch.zeros(1, 3, 2, 16, 64), v_pool=torch.zeros(1, 3, 2, 16, 64))),
    ("tree_attention", dict(max_nodes=0)),
    ("tree_attention", dict(max_nodes=513)),
    ("tree_attention", dict(max_nodes=65)),  # more than the mask's bits
    ("tree_attention", dict(mask=torch.zeros(4, 1, dtype=I64))),
    ("tree_attention", dict(mask=torch.zeros(5, 1, dtype=I32))),
    ("tree_attention", dict(mask=torch.zeros(5, 2, dtype=I64)[:, :1])),
    ("tree_attention", dict(cu_nodes=torch.tensor([0, 2, 5], dtype=I32))),
    ("tree_attention", dict(lengths=torch.ones(1, dtype=I64))),
    ("tree_attention", dict(scale=0.0)),
    ("tree_attention", dict(scale=-1.0)),
    ("tree_attention", dict(scale=float("nan"))),
    ("tree_attention", dict(scale=float("inf"))),
    ("tree_attention", dict(out=torch.zeros(5, 4, 32))),
    ("tree_attention", dict(out=torch.zeros(5, 4, 64), out_dtype=torch.float16)),
    ("tree_attention", dict(q=_q, out=_q)),
    ("tree_attention", dict(out=torch.zeros(1, 4, 64).expand(5, 4, 64))),
    ("tree_attention", dict(out=torch.zeros(5, 1, 64).expand(5, 4, 64))),
    ("tree_attention", dict(lse=torch.zeros(4, 5))),
    ("tree_attention", dict(k_pool=_same, v_pool=torch.zeros(3, 2, 16, 64), lse=_same.view(-1)[:20].view(5, 4))),
    ("tree_attention", dict(k_pool=torch.zeros(3, 2, 16, 64), v_pool=_same, lse=_same.view(-1)[:20].view(5, 4))),
    ("tree_attention", dict(q=_q, lse=_q.view(-1)[:20].view(5, 4))),
    ("tree_attention", dict(out=_out, lse=_out.view(-1)[:20].view(5, 4))),
    ("commit_path", dict(path=torch.zeros(2, 65, dtype=I32))),
    ("commit_path", dict(path=torch.zeros(2, 0, dtype=I32))),
    ("commit_path", dict(path=torch.zeros(8, dtype=I32))),
    ("commit_path", dict(path=torch.zeros(2, 8, dtype=I32)[:, ::2])),
    ("commit_path", dict(n_path=torch.ones(2, dtype=I64))),
    ("commit_path", dict(block_table=torch.zeros(1, 3, dtype=I32))),
    ("commit_path", dict(lengths=_lengths, out=_lengths)),
    ("commit_path", dict(out=torch.ones(3, dtype=I32))),
    ("commit_path", dict(path=_path, out=_path.view(-1))),
    ("commit_path", dict(n_path=_lengths, out=_lengths)),
    ("commit_path", dict(k_pool=_same, v_pool=_same)),
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
    assert [c[0] for c in lib.calls] == ["halo_" + ("tree_attn" if name == "tree_attention" else name)]


@pytest.mark.parametrize("name", CALLS)
def test_tensors_on_the_host_are_refused(monkeypatch, name):
    from halo_amd import block_pool
    import halo_amd
    lib = _Lib()
    monkeypatch.setattr(block_pool.nat, "lib", lambda: lib)
    with pytest.raises(AssertionError, match="GPU"):
        getattr(halo_amd, name)(**CALLS[name]())
    assert lib.calls == []


def test_pool_record(lib):
    from halo_amd.block_pool import pack_pool
    k = torch.zeros(2, 7, 3, 16, 64, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    f = struct.unpack("<2Q4q6i", pack_pool(k, v))
    assert f == (k.data_ptr(), v.data_ptr(), 7 * 3 * 16 * 64, 3 * 16 * 64, 16 * 64, 64, 2, 7, 3, 16, 64, 1)
    f = struct.unpack("<2Q4q6i", pack_pool(k[1].transpose(1, 2).contiguous().transpose(1, 2),
                                           v[0].transpose(1, 2).contiguous().transpose(1, 2)))
    assert f[2:] == (0, 3 * 16 * 64, 64, 3 * 64, 1, 7, 3, 16, 64, 1)


def test_calls_without_nodes_or_rows_do_not_launch(lib):
    import halo_amd
    halo_amd.tree_layout(torch.zeros(0, dtype=I32), torch.zeros(2, dtype=I32), max_nodes=4)
    assert lib.calls == []


# ---------------------------------------------------------------- the C entries' own checks

@pytest.fixture
def entries():
    from halo_amd import _native as nat
    if not nat.loadable():
        pytest.skip("library not built (run __graft_entry__.build())")
    if torch.cuda.is_available():
        pytest.skip("these calls must not reach a GPU")
    return nat._load()


def _pool(**kw):
    """A pool record whose pointers are never followed: the calls are refused before."""
    d = dict(k=4096, v=8192, sl=0, sb=2048, sh=1024, sr=64, layers=1, blocks=3, H_kv=2, bs=16, D=64, dt=1)
    d.update(kw)
    return struct.pack("<2Q4q6i", *d.values())


def _attn(lib, pool=None, **kw):
    d = dict(q=4096, qn=256, qh=64, N=5, H=4, table=4096, ts=3, B=1, W=3, lengths=4096, cu=4096, max_nodes=5, mask=None,
             ms=0, scale=0.125, out=4096, on=256, oh=64, odt=1, lse=None, ws=None, nb=0, st=None)
    d.update(kw)
    return lib.halo_tree_attn(pool or _pool(), *d.values())


@pytest.mark.parametrize("kw", [
    dict(pool=_pool(dt=3)), dict(pool=_pool(D=96)), dict(pool=_pool(layers=2)), dict(pool=_pool(k=0)),
    dict(pool=_pool(k=4104)), dict(pool=_pool(sr=68)), dict(pool=_pool(sb=-2048)), dict(pool=_pool(bs=0)),
    dict(pool=_pool(blocks=2 ** 31 - 1, sb=2 ** 40)), dict(H=5), dict(H=0), dict(B=0), dict(W=0), dict(max_nodes=0),
    dict(max_nodes=513), dict(q=4100), dict(q=None), dict(qn=257), dict(table=None), dict(ts=2), dict(W=2 ** 28, ts=2 ** 28),
    dict(mask=4096, ms=0), dict(scale=0.0), dict(scale=float("nan")), dict(scale=1e-42), dict(out=None), dict(odt=7), dict(odt=2), dict(out=4100), dict(on=258), dict(oh=65),
    dict(N=-1), dict(W=3000, ts=3000)])
def test_tree_attn_entry_refuses(entries, kw):
    assert _attn(entries, **kw) == -1
    assert entries.halo_last_error()


def test_tree_attn_entry_wants_its_workspace(entries):
    need = entries.halo_tree_workspace_size(1, 1, 4, 2, 64, 3000 * 16, 5)
    assert need > 0
    assert _attn(entries, W=3000, ts=3000, ws=4096, nb=need - 1) == -4
    assert _attn(entries, W=3000, ts=3000, ws=4100, nb=need) == -1


def test_other_entries_refuse(entries):
    p = 4096
    upd = lambda **kw: entries.halo_update_block_tables(*{**dict(t=p, ts=4, n=p, B=2, W=4, f=p, cap=9, nf=p, ln=p, fi=p,  # noqa: E731
                                                                 bs=16, mr=4, cu=p, sl=p, ok=p, st=None), **kw}.values())
    for kw in (dict(t=None), dict(B=0), dict(W=0), dict(ts=3), dict(bs=0), dict(mr=-1), dict(sl=None), dict(cap=-1),
               dict(W=2 ** 30, ts=2 ** 30)):
        assert upd(**kw) == -1
    app = lambda pool=_pool(), **kw: entries.halo_append_rows(pool, *{**dict(k=p, kl=0, kn=128, kh=64, v=p, vl=0, vn=128,  # noqa: E731
                                                                             vh=64, s=p, N=5, st=None), **kw}.values())
    for kw in (dict(k=None), dict(s=None), dict(N=-1), dict(pool=_pool(dt=9)), dict(pool=_pool(blocks=0)),
               dict(pool=_pool(blocks=2 ** 30, bs=4)), dict(pool=_pool(layers=70000))):
        assert app(**kw) == -1
    lay = lambda **kw: entries.halo_tree_layout(*{**dict(pa=p, cu=p, B=1, N=5, mn=5, m=p, ms=1, d=p, st=None), **kw}.values())  # noqa: E731
    for kw in (dict(pa=None), dict(B=0), dict(N=0), dict(mn=0), dict(mn=513), dict(mn=65)):
        assert lay(**kw) == -1
    com = lambda pool=_pool(), **kw: entries.halo_commit_path(pool, *{**dict(t=p, ts=4, B=1, W=4, ln=p, pa=p, ps=4, P=4, n=p,  # noqa: E731
                                                                             new=2 * p, st=None), **kw}.values())
    for kw in (dict(t=None), dict(B=0), dict(B=70000), dict(P=65), dict(P=0), dict(new=p), dict(pool=_pool(D=0))):
        assert com(**kw) == -1


def test_pool_struct_size():
    class P(ctypes.Structure):
        _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in "lbhr"] + \
                   [(n, ctypes.c_int32) for n in ("layers", "blocks", "H", "bs", "D", "dt")]
    assert ctypes.sizeof(P) == 72
