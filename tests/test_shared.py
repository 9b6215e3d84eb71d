"""Attention behind shared prefixes on the CPU: argument checks before any launch."""

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


def _plan(L, table=P, W=4, R=2, NG=1, T=3, H=4, HK=2, D=64, page=16, schedule=P, ints=1 << 30):
    return L.mi_paged_shared_plan(table, W, P, P, R, P, NG, T, H, HK, D, page, P, schedule, ints, None)


def _attn(L, q=P, out=P, schedule=P, W=4, R=2, NG=1, T=3, H=4, HK=2, D=64, pages=8, page=16,
          dt=hip.MI_BF16, ws=P, nbytes=1 << 40):
    return L.mi_paged_shared_attention(q, P, P, out, P, schedule, T, R, NG, W, H, HK, D, pages, page,
                                       0.1, dt, ws, nbytes, None)


@pytest.mark.parametrize("call", [_plan, _attn])
@pytest.mark.parametrize("kw,code,text", [
    ({"D": 96}, 2, b"head dim 96"), ({"page": 20}, 2, b"page size 20"), ({"T": -1}, 1, b"T=-1"),
    ({"T": (1 << 18) + 1}, 1, b"T=262145"), ({"R": 0}, 1, b"R=0"), ({"R": 4097}, 1, b"R=4097"),
    ({"NG": 0}, 1, b"groups=0"), ({"NG": 3}, 1, b"groups=3"), ({"W": 0}, 1, b"width 0"),
    ({"H": 5}, 1, b"H=5"), ({"HK": 0}, 1, b"HK=0"), ({"schedule": None}, 1, b"null"),
    ({"schedule": P + 4}, 1, b"aligned"),
])
def test_refusals(lib, call, kw, code, text):
    assert call(lib, **kw) == code
    assert text in lib.mi_last_error()


@pytest.mark.parametrize("kw,code,text", [
    ({"dt": hip.MI_F32}, 2, b"bf16 and fp16"), ({"pages": 0}, 1, b"pages=0"),
    ({"q": P + 8}, 1, b"aligned"), ({"out": P + 4}, 1, b"aligned"), ({"q": None}, 1, b"null"),
    ({"ws": None}, 1, b"workspace"), ({"ws": P + 8}, 1, b"workspace"), ({"nbytes": 64}, 1, b"workspace"),
])
def test_attention_refusals(lib, kw, code, text):
    assert _attn(lib, **kw) == code
    assert text in lib.mi_last_error()


def test_plan_refusals(lib):
    assert _plan(lib, table=None) == 1 and b"null" in lib.mi_last_error()
    assert _plan(lib, ints=10) == 1 and b"ints" in lib.mi_last_error()
    assert _plan(lib, T=(1 << 18) - 1, R=4096, NG=4096, H=16, HK=1) == 1
    assert b"at most 65535" in lib.mi_last_error()
    assert lib.mi_paged_shared_plan_ints(3, 2, 3, 4, 4, 2, 64, 16) == 0
    assert _attn(lib, T=0) == 0


def _arrays():
    i = dict(dtype=torch.int32)
    return dict(block_table=torch.zeros((2, 3), **i), cu_q=torch.zeros(3, **i),
                kv_lens=torch.zeros(2, **i), cu_groups=torch.zeros(2, **i))


SIZES = dict(page_size=16, num_tokens=2, n_heads=4, n_kv_heads=2, head_dim=64)


def test_ops_refuse():
    a = _arrays()
    with pytest.raises(RuntimeError):
        ops.paged_shared_plan(**a, **SIZES)
    i = a["kv_lens"]
    for bad in (dict(block_table=a["block_table"][0]), dict(block_table=a["block_table"][:1]),
                dict(cu_q=i), dict(cu_groups=i[:1]), dict(cu_groups=i.long()), dict(kv_lens=i.long()),
                dict(block_table=torch.zeros((3, 2), dtype=torch.int32).t())):
        with pytest.raises(ValueError):
            ops.paged_shared_plan(**{**a, **bad}, **SIZES)


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks alone are run."""
    is_cuda = True


def test_ops_refuse_other_sizes(monkeypatch):
    for name in ("paged_shared_plan", "paged_shared_attention"):
        monkeypatch.setattr(hip, name, lambda *a: pytest.fail("launched"))
    a = _arrays()
    a["block_table"] = a["block_table"].as_subclass(_Gpu)
    for bad in (dict(page_size=24), dict(n_heads=5), dict(head_dim=80), dict(num_tokens=-1)):
        with pytest.raises(ValueError):
            ops.paged_shared_plan(**a, **{**SIZES, **bad})
    shape = (2, 2, 1, 3, 4, 2, 64, 16)
    plan = ops.SharedPlan(a["kv_lens"][:1], torch.zeros(99, dtype=torch.int32), shape)
    for i in (0, 3, 4, 7):
        other = plan._replace(shape=shape[:i] + (shape[i] * 2,) + shape[i + 1:])
        with pytest.raises(ValueError):
            ops.paged_shared_plan(**a, **SIZES, out=other)
    q, pool = torch.zeros((2, 4, 64), dtype=torch.bfloat16), torch.zeros((8, 2, 16, 64), dtype=torch.bfloat16)
    kw = dict(q=q, k_pages=pool, v_pages=pool, block_table=_arrays()["block_table"], plan=plan, scale=1.0)
    for bad in (dict(q=q[:1]), dict(q=q.half()), dict(q=q[:, :2]), dict(k_pages=pool[:4]),
                dict(k_pages=pool[:, :1], v_pages=pool[:, :1]), dict(block_table=kw["block_table"][:1]),
                dict(block_table=kw["block_table"].long()),
                dict(k_pages=pool.view(4, 2, 32, 64), v_pages=pool.view(4, 2, 32, 64))):
        with pytest.raises(ValueError):
            ops.paged_shared_attention(**{**kw, **bad})
