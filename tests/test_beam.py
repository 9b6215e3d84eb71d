"""Beam selection on the CPU: argument checks before any launch."""

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


def _select(L, x=P, stride=100, scores=P, finished=None, eos=-1, R=2, B=3, V=100, K=3, out=P,
            dt=hip.MI_BF16, ws=P, nbytes=1 << 30):
    return L.mi_beam_select(x, stride, scores, finished, eos, R, B, V, K, out, P, P, P, dt, ws, nbytes,
                            None)


@pytest.mark.parametrize("kw,code,text", [
    ({"dt": 7}, 2, b"dtype code 7"), ({"R": -1}, 1, b"R=-1"), ({"R": 4097}, 1, b"R=4097"),
    ({"B": 0}, 1, b"B=0"), ({"B": 65}, 1, b"B=65"), ({"V": 0}, 1, b"V=0"),
    ({"V": (1 << 20) + 1}, 1, b"V=1048577"), ({"stride": -1}, 1, b"stride -1"),
    ({"K": 0}, 1, b"K=0"), ({"K": 65}, 1, b"K=65"), ({"K": 7, "V": 2}, 1, b"K=7"),
    ({"eos": 100}, 1, b"eos=100"), ({"eos": -2}, 1, b"eos=-2"), ({"finished": P}, 1, b"eos=-1"),
    ({"x": None}, 1, b"null"), ({"scores": None}, 1, b"null"), ({"out": None}, 1, b"null"),
    ({"x": P + 1}, 1, b"aligned"), ({"ws": None}, 1, b"workspace"), ({"ws": P + 8}, 1, b"workspace"),
    ({"nbytes": 100}, 1, b"workspace"),
])
def test_refusals(lib, kw, code, text):
    assert _select(lib, **kw) == code
    assert text in lib.mi_last_error()


def test_of_no_prompts(lib):
    assert _select(lib, R=0, ws=None, nbytes=0) == 0
    assert lib.mi_beam_select_workspace_bytes(0, 4, 100, 4) == 0


def test_workspace_covers_every_row(lib):
    """The prefix of tickets, and at least a list and a sum a row."""
    for R, B, V, K in ((1, 1, 1, 1), (1, 4, 151936, 4), (511, 1, 65537, 64), (512, 1, 5, 3),
                       (4096, 64, 1 << 20, 64)):
        n = lib.mi_beam_select_workspace_bytes(R, B, V, K)
        assert n >= 18432 + R * B * (8 + 8 * K)


def test_ops_refuse():
    x, s = torch.zeros(6, 50, dtype=torch.bfloat16), torch.zeros(2, 3)
    with pytest.raises(RuntimeError):
        ops.beam_select(x, s)


class _Gpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks alone are run."""
    is_cuda = True


def test_ops_refuse_wrong_arrays(monkeypatch):
    monkeypatch.setattr(hip, "beam_select", lambda *a: pytest.fail("launched"))
    x = torch.zeros(6, 50, dtype=torch.bfloat16).as_subclass(_Gpu)
    s, f = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.bool)
    for bad in (dict(scores=s.double()), dict(scores=s[0]), dict(scores=s.t()), dict(logits=x[:5]),
                dict(logits=x[None]), dict(finished=f), dict(finished=f[:1], eos=1),
                dict(finished=f.byte(), eos=1), dict(finished=f.t(), eos=1), dict(width=0),
                dict(width=-3)):
        with pytest.raises(ValueError):
            ops.beam_select(**{**dict(logits=x, scores=s), **bad})
