"""The paged-cache entries and the log probabilities on the CPU: argument checks
before any launch, the step plan's definition, the rotation table."""

from __future__ import annotations

import ctypes
import math

import numpy as np
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


def _plan(L, table=P, width=4, R=2, T=3, page=16, n_free=8):
    return L.mi_paged_plan(table, width, P, P, P, n_free, P, R, T, page, P, P, P, P, P, P, None)


@pytest.mark.parametrize("kw,code,text", [
    ({"page": 8}, 2, b"page size 8"), ({"page": 48}, 2, b"page size 48"),
    ({"page": 512}, 2, b"page size 512"), ({"R": 0}, 1, b"R=0"), ({"R": 4097}, 1, b"R=4097"),
    ({"width": 0}, 1, b"table width 0"), ({"width": 131073}, 1, b"131073"),
    ({"T": -1}, 1, b"T=-1"), ({"table": None}, 1, b"null"), ({"n_free": -1}, 1, b"free pages -1"),
    ({"T": 262145}, 1, b"T=262145"),
])
def test_plan_refusals(lib, kw, code, text):
    assert _plan(lib, **kw) == code
    assert text in lib.mi_last_error()


def _rope(L, q=P, stride=256, qn=P, dims=128, T=2, Hq=2, Hkv=1, D=128, pages=4, page=16,
          dt=hip.MI_BF16, table=P):
    return L.mi_norm_rope_paged(q, P, P, stride, 128, 128, qn, P, P, P, P, table, dims, 0, P, P, T,
                                Hq, Hkv, D, pages, page, 1e-6, dt, None)


@pytest.mark.parametrize("kw,code,text", [
    ({"dt": hip.MI_F32}, 2, b"bf16 and fp16"), ({"D": 96}, 2, b"head dim 96"),
    ({"page": 24}, 2, b"page size 24"), ({"dims": 12}, 1, b"rope dims 12"),
    ({"dims": 136}, 1, b"rope dims 136"), ({"dims": -8}, 1, b"rope dims -8"),
    ({"stride": 257}, 1, b"aligned"), ({"q": P + 8}, 1, b"aligned"), ({"qn": P + 4}, 1, b"aligned"),
    ({"q": None}, 1, b"null"), ({"table": None}, 1, b"null"), ({"pages": 0}, 1, b"pages=0"),
    ({"pages": 1 << 27}, 1, b"2^31"), ({"T": -1}, 1, b"T=-1"), ({"Hkv": 0}, 1, b"Hkv=0"),
])
def test_prologue_refusals(lib, kw, code, text):
    assert _rope(lib, **kw) == code
    assert text in lib.mi_last_error()


def test_prologue_of_no_tokens(lib):
    assert _rope(lib, T=0) == 0


def _attn(L, q=P, T=2, R=2, W=4, H=4, HK=2, D=128, pages=8, page=16, dt=hip.MI_BF16, out=P):
    return L.mi_paged_attention(q, P, P, out, P, P, P, T, R, W, H, HK, D, pages, page, 0, 0.1, dt,
                                None, 0, None)


@pytest.mark.parametrize("kw,code,text", [
    ({"dt": hip.MI_F32}, 2, b"bf16 and fp16"), ({"D": 80}, 2, b"head dim 80"),
    ({"page": 20}, 2, b"page size 20"), ({"H": 5}, 1, b"H=5"), ({"HK": 0}, 1, b"HK=0"),
    ({"T": -1}, 1, b"T=-1"), ({"R": -1}, 1, b"R=-1"), ({"W": 0}, 1, b"table width 0"),
    ({"pages": 0}, 1, b"pages=0"), ({"q": P + 8}, 1, b"aligned"), ({"out": P + 4}, 1, b"aligned"),
    ({"q": None}, 1, b"null"),
])
def test_attention_refusals(lib, kw, code, text):
    assert _attn(lib, **kw) == code
    assert text in lib.mi_last_error()


def test_attention_of_nothing(lib):
    assert _attn(lib, T=0) == 0 and _attn(lib, R=0) == 0


def _lp(L, x=P, rows=2, V=100, stride=100, tokens=P, top=5, dt=hip.MI_BF16, ids=P):
    return L.mi_token_logprobs(x, rows, V, stride, tokens, 1, top, P, P, ids, P, dt, None, 0,
                               None)


@pytest.mark.parametrize("kw,code,text", [
    ({"dt": 7}, 2, b"dtype code 7"), ({"V": 0}, 1, b"V=0"), ({"rows": -1}, 1, b"rows=-1"),
    ({"top": -1}, 1, b"top=-1"), ({"top": 65}, 1, b"top=65"), ({"top": 7, "V": 6}, 1, b"V=6"),
    ({"tokens": None}, 1, b"null"), ({"ids": None}, 1, b"null"), ({"x": P + 1}, 1, b"aligned"),
    ({"stride": -1}, 1, b"stride -1"),
])
def test_logprob_refusals(lib, kw, code, text):
    assert _lp(lib, **kw) == code
    assert text in lib.mi_last_error()


def test_logprobs_of_no_rows(lib):
    assert _lp(lib, rows=0) == 0


def test_ops_refuse_cpu_tensors():
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    pages = torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.paged_plan(i[None], i, i, i, i, 16, 1)
    with pytest.raises(RuntimeError):
        ops.norm_rope_paged(x, x, x, None, None, 1, 1, 1e-6, ops.rope_table(64, device="cpu"), i, i,
                            pages, pages)
    with pytest.raises(RuntimeError):
        ops.paged_attention(x[:, None], pages, pages, i[None], torch.zeros(2, dtype=torch.int32), i, 1.0)
    with pytest.raises(RuntimeError):
        ops.token_logprobs(x, i)


def test_ops_refuse_wrong_arrays():
    """The checks of shapes and types, which come before the device's."""
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    pages = torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16)
    t = ops.rope_table(64, device="cpu")
    cu = torch.zeros(2, dtype=torch.int32)
    for bad in (dict(k=x[:, :64]), dict(positions=i.long()), dict(slots=cu), dict(inv_freq=t.float()),
                dict(q_norm=x[0].float()), dict(k_pages=pages.half()), dict(k_pages=pages[..., :64]),
                dict(n_kv_heads=2)):
        kw = dict(q=x, k=x, v=x, q_norm=None, k_norm=None, n_heads=1, n_kv_heads=1, eps=1e-6,
                  inv_freq=t, positions=i, slots=i, k_pages=pages, v_pages=pages)
        with pytest.raises(ValueError):
            ops.norm_rope_paged(**{**kw, **bad})
    for bad in (dict(q=x), dict(cu_q=i), dict(kv_lens=i.long()), dict(block_table=i),
                dict(v_pages=pages[:1]), dict(k_pages=pages.transpose(1, 2))):
        kw = dict(q=x[:, None], k_pages=pages, v_pages=pages, block_table=i[None], cu_q=cu,
                  kv_lens=i, scale=1.0)
        with pytest.raises(ValueError):
            ops.paged_attention(**{**kw, **bad})


def test_launches_happen_on_the_tensors_device(monkeypatch):
    """Where the current device is another one, it is changed for the launch."""
    seen = []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            seen.append(self.index)

        def __exit__(self, *a):
            seen.append("back")

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    with ops._on(1):
        seen.append("launch")
    with ops._on(0):
        seen.append("here")
    assert seen == [1, "launch", "back", "here"]


def test_rope_table():
    t = ops.rope_table(64, 1e6, device="cpu")
    want = np.array([1e6 ** (-2 * i / 64) for i in range(32)])
    assert t.dtype == torch.float64 and np.abs(t.numpy() / want - 1).max() < 1e-14
    assert torch.equal(ops.rope_table(64, 1e6, 0.25, device="cpu"), t * 0.25)
    f = torch.tensor([1.0, 3.0, 700.0, 1e5])
    assert torch.equal(ops.rope_table(8, freqs=f, device="cpu"), 1 / f.double())
    with pytest.raises(ValueError):
        ops.rope_table(16, freqs=f, device="cpu")
    assert ops.rope_table(0, device="cpu").numel() == 0
    assert math.isclose(float(ops.rope_table(8, 1e4, device="cpu")[1]), 0.1)
