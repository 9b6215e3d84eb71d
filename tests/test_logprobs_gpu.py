"""Token log probabilities, entropies and top tokens against float64."""

from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402

DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def reference(x, tokens, top):
    """float64 numpy: (logprobs, entropy, ids, top logprobs); ids by (value
    descending, index ascending). (x - m) - log S, not x - (m + log S): at a mask's
    3e38 float64 would lose log S."""
    y = x.double().cpu().numpy()
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = y.max(-1, keepdims=True)
        e = np.exp(y - m)
        S = e.sum(-1, keepdims=True)
        y0 = (y - m) - np.log(S)
        ent = np.log(S)[:, 0] - np.where(e > 0, e * (y - m), 0).sum(-1) / S[:, 0]
        ids = np.argsort(-y, axis=-1, kind="stable")[:, :top]
        lp = np.take_along_axis(y0, tokens.cpu().numpy().astype(np.int64)[:, None], 1)[:, 0]
        return lp, ent, ids, np.take_along_axis(y0, ids, 1)


def check(x, tokens, top):
    """fp32 sums of V terms, each lane's share (V / 256 and a few more) added in
    turn: log S errs by that many times 2^-24, and as much for the exponentials
    (2^-23 of a term, and 2^-24 of its exponent, at most 104 log2 e, weighted by a
    term that is 2^-exponent: under 2^-23 in all); the difference x - m - log S by
    two roundings of its size. The entropy's quotient errs by twice as much of
    itself."""
    lp, ent, ids, tlp = reference(x, tokens, top)
    r = ops.token_logprobs(x, tokens, top)
    n = (x.shape[-1] / 256 + 40) * 2.0 ** -24
    for got, want in ((r.logprobs, lp), (r.top_logprobs, tlp)):
        got = got.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isneginf(got), np.isneginf(want))
        fine = np.isfinite(want)
        assert (np.abs(got[fine] - want[fine]) <= n + 2.0 ** -22 * np.abs(want[fine])).all()
    e = r.entropy.cpu().numpy().astype(np.float64)
    assert (np.abs(e - ent) <= 3 * n * (1 + np.abs(ent))).all(), np.abs(e - ent).max()
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    assert r.logprobs.dtype == F32 and r.top_ids.dtype == torch.int32
    return r


def logits(seed, rows, V, dtype, spread=3.0, masked=0.0):
    g = torch.Generator()
    g.manual_seed(seed)
    x = spread * torch.randn((rows, V), generator=g)
    if masked:
        x[torch.rand((rows, V), generator=g) < masked] = -math.inf
        x[:, V // 2] = 1.0
    return x.to(dtype).to(DEV), torch.randint(0, V, (rows,), generator=g).to(DEV)


@pytest.mark.parametrize("rows,V,dtype,top,spread,masked", [
    (1, 1, BF, 1, 1, 0), (3, 2, F32, 2, 1, 0), (2, 7, FP, 5, 3, 0), (5, 64, BF, 64, 3, 0),
    (4, 255, BF, 20, 3, 0), (3, 256, F32, 1, 3, 0), (2, 257, FP, 33, 3, 0), (3, 2047, BF, 0, 3, 0),
    (2, 2049, BF, 64, 0.01, 0),           # many ties
    (7, 4099, FP, 20, 3, 0.9), (3, 5000, F32, 5, 30, 0.5), (1, 151936, BF, 5, 3, 0),
    (9, 65537, FP, 20, 3, 0.9), (2, 128257, F32, 20, 1, 0), (40, 32000, BF, 1, 3, 0),
    (300, 1000, BF, 8, 3, 0), (3, 40000, BF, 64, 0, 0),      # all equal
    (2, 3000, BF, 20, 3, 0.998),          # fewer finite logits than top: -inf, lowest index first
    (2, 70000, FP, 64, 3, 0.9999),
])
def test_logprobs(rows, V, dtype, top, spread, masked):
    check(*logits(rows + V, rows, V, dtype, spread, masked), top)


@pytest.mark.parametrize("top", [1, 20, 64])
def test_orders(top):
    """Ascending, descending, largest at the ends, far above or below zero."""
    V = 9001
    up = torch.arange(V, dtype=F32) / 100
    rows = [up, up.flip(0), -up.abs() - 1e4, up + 1e4, torch.zeros(V), torch.zeros(V)]
    rows[4][V - 1] = 60.0
    rows[5][0] = 60.0
    x = torch.stack(rows).to(DEV)
    tok = torch.tensor([0, 1, V - 1, 5, V - 1, 0], device=DEV)
    # up + 1e4: neighbours' gaps of 0.01 are 10 steps of fp32, their own roundings the input's
    check(x, tok, top)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_lowest_values(dtype):
    """A mask of the type's lowest value, and a row of nothing else."""
    V, low = 3001, torch.finfo(dtype).min
    x = torch.full((2, V), low, dtype=dtype, device=DEV)
    x[0, 100], x[0, 2000] = 1.0, 2.0
    r = check(x, torch.tensor([2000, 17], device=DEV), 4)
    assert r.top_ids.tolist() == [[2000, 100, 0, 1], [0, 1, 2, 3]]
    assert abs(float(r.entropy[1]) - math.log(V)) < 1e-5


def test_strides_and_shapes():
    """Rows of odd lengths (16-byte pieces that begin before them), a last-position
    view, leading axes, int32 tokens, repeated rows."""
    x, _ = logits(5, 12, 3001, BF)
    tok = torch.arange(12, device=DEV, dtype=torch.int32)
    a = check(x, tok, 3)
    cube, tk = x.view(4, 3, 3001), tok.view(4, 3)
    b = ops.token_logprobs(cube, tk, 3)
    assert b.logprobs.shape == (4, 3) and b.top_ids.shape == (4, 3, 3)
    assert all(torch.equal(s.flatten(), t.flatten()) for s, t in zip(a, b))
    check(cube[:, -1, :], tk[:, -1], 3)
    check(x[:, 5:2000], tok, 7)
    check(x[:, :3000:3].contiguous(), tok, 7)
    t = ops.token_logprobs(x.t().contiguous().t(), tok, 3)
    assert all(torch.equal(s, u) for s, u in zip(a, t))
    e = ops.token_logprobs(x[:1].expand(5, -1), tok[:5], 2)
    assert all(torch.equal(e.entropy[0], v) for v in e.entropy)
    z = ops.token_logprobs(x[:0], tok[:0], 2)
    assert z.logprobs.shape == (0,) and z.top_ids.shape == (0, 2)
    one = ops.token_logprobs(x[0], tok[0], 2)
    assert one.logprobs.shape == () and one.top_ids.tolist() == a.top_ids[0, :2].tolist()


def test_no_answer_is_nan():
    """Tokens outside the vocabulary; rows with NaN, +inf, or -inf alone. The rows
    beside them are not touched."""
    x, tok = logits(6, 6, 4097, BF)
    want = ops.token_logprobs(x, tok, 4)
    bad, t = x.clone(), tok.clone()
    bad[1, 4000], bad[2, 3], t[3], t[5] = math.nan, math.inf, -1, 4097
    bad[4] = -math.inf
    r = ops.token_logprobs(bad, t, 4)
    assert r.logprobs.isnan().tolist() == [False, True, True, True, True, True]
    assert r.entropy.isnan().tolist() == [False, True, True, False, True, False]
    assert bool((r.top_ids >= 0).all()) and bool((r.top_ids < 4097).all())
    for i in (0, 3, 5):
        assert torch.equal(r.entropy[i], want.entropy[i]) and torch.equal(r.top_ids[i], want.top_ids[i])
    assert torch.equal(r.logprobs[0], want.logprobs[0])


def test_without_a_workspace(monkeypatch):
    """The C entry without scratch: a workgroup a row, the same answers."""
    from autotuner_runtime import hip

    x, tok = logits(8, 3, 40001, BF)
    want = check(x, tok, 7)
    need = hip._logprobs_workspace_bytes
    for short in (lambda *a: 0, lambda *a: need(*a) - 1):
        monkeypatch.setattr(hip, "_logprobs_workspace_bytes", short)
        got = check(x, tok, 7)
        assert torch.equal(got.top_ids, want.top_ids)


def test_repeats_and_graphs():
    """The same bits from call to call, and from a graph replayed over new logits."""
    from autotuner_runtime import hip

    x, tok = logits(9, 3, 65537, BF)
    y, _ = logits(10, 3, 65537, BF)
    want = [ops.token_logprobs(v, tok, 5) for v in (x, y)]
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with hip.graph_workspaces(), torch.cuda.graph(graph):
        out = ops.token_logprobs(static, tok, 5)
    for i in (0, 1, 1, 0, 1):
        static.copy_((x, y)[i])
        ops.token_logprobs(y, tok, 5)  # eager work between
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i


def test_refusals():
    x, tok = logits(7, 3, 100, BF)
    for top in (-1, 65, 101):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, tok, top)
    for bad in (tok[:2], tok.float(), tok[:, None], tok.cpu()):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, bad, 1)
    with pytest.raises(ValueError):
        ops.token_logprobs(x.double(), tok, 1)
