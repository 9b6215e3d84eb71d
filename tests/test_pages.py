"""Forking and compacting pages on the CPU: argument checks before any launch."""

from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")
from autotuner_runtime import hip, ops  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    L = ctypes.CDLL(str(hip.library_path()))
    for name, args in hip.SIGNATURES.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = hip.RESTYPES.get(name, ctypes.c_int)
    return L


P = 0x1000  # a 16-byte aligned address that is never read


def _fork(L, table=P, W=4, R=2, n_free=8, pools=P, n_pools=2, pages=8, HK=2, page=16, row=128, ws=P,
          nbytes=1 << 30):
    return L.mi_paged_fork(table, W, P, P, R, P, n_free, P, P, pools, n_pools, pages, HK, page, row,
                           ws, nbytes, None)


def _compact(L, table=P, W=4, R=2, n_free=8, pools=P, n_pools=2, pages=8, HK=2, page=16, row=128,
             ws=P, nbytes=1 << 30):
    return L.mi_paged_compact(table, W, P, R, P, n_free, P, P, pools, n_pools, pages, HK, page, row,
                              ws, nbytes, None)


@pytest.mark.parametrize("call", [_fork, _compact])
@pytest.mark.parametrize("kw,code,text", [
    ({"page": 8}, 2, b"page size 8"), ({"page": 48}, 2, b"page size 48"),
    ({"page": 512}, 2, b"page size 512"), ({"R": 0}, 1, b"R=0"), ({"R": -1}, 1, b"R=-1"),
    ({"R": 4097}, 1, b"R=4097"), ({"W": 0}, 1, b"table width 0"), ({"W": 131073}, 1, b"131073"),
    ({"pages": 0}, 1, b"pages=0"), ({"pages": (1 << 20) + 1, "n_free": 1 << 21}, 1, b"pages=1048577"),
    ({"n_free": 7}, 1, b"free list of 7"), ({"n_pools": -1}, 1, b"pools=-1"),
    ({"n_pools": 65537}, 1, b"pools=65537"), ({"HK": 0}, 1, b"heads=0"), ({"row": 0}, 1, b"rows of 0"),
    ({"row": 24}, 1, b"rows of 24"), ({"table": None}, 1, b"null"), ({"pools": None}, 1, b"null"),
    ({"ws": None}, 1, b"workspace"), ({"ws": P + 8}, 1, b"workspace"), ({"nbytes": 1000}, 1, b"workspace"),
])
def test_refusals(lib, call, kw, code, text):
    assert call(lib, **kw) == code
    assert text in lib.mi_last_error()


def _arrays(device="cpu"):
    i32 = dict(dtype=torch.int32, device=device)
    return dict(block_table=torch.zeros((2, 3), **i32), kv_lens=torch.zeros(2, **i32),
                free_pages=torch.zeros(8, **i32), free_count=torch.zeros(1, **i32))


def _pools():
    p = torch.zeros((8, 2, 16, 64), dtype=torch.bfloat16)
    return ops.PagePools(torch.zeros(1, dtype=torch.int64), (p,), (8, 2, 16, 128))


def test_pools_refuse():
    p = torch.zeros((8, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.page_pools([])
    with pytest.raises(RuntimeError):
        ops.page_pools([p])


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks alone are run."""
    is_cuda = True


def test_pools_refuse_wrong_arrays():
    p = torch.zeros((8, 2, 16, 64), dtype=torch.bfloat16).as_subclass(_Gpu)
    for bad in (p[:4], p.half(), p.transpose(1, 2), p[..., :32], p[0]):
        with pytest.raises(ValueError):
            ops.page_pools([p, bad])


def test_ops_refuse_wrong_arrays(monkeypatch):
    monkeypatch.setattr(hip, "paged_fork", lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(hip, "paged_compact", lambda *a: pytest.fail("launched"))
    a = _arrays()
    s = torch.zeros(2, dtype=torch.int32)
    wrong = (dict(block_table=a["block_table"][0]), dict(kv_lens=s[:1]), dict(kv_lens=s.long()),
             dict(free_count=s), dict(free_pages=s.view(1, 2)), dict(block_table=a["block_table"].t()),
             dict(block_table=torch.zeros((0, 3), dtype=torch.int32), kv_lens=s[:0]))
    for bad in wrong:
        with pytest.raises(ValueError):
            ops.paged_compact(**{**a, **bad}, pools=_pools())
    for bad in (*wrong, dict(sources=s[:1]), dict(sources=s.long())):
        with pytest.raises(ValueError):
            ops.paged_fork(**{**a, "sources": s, **bad}, pools=_pools())
