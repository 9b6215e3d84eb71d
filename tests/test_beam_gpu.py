"""Beam selection against its definition in 64 bits."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import hip, ops  # noqa: E402

DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
# A row's lse: a lane adds 16 values of a chunk one after another, then at most 128 chunks;
# eight waves' sums, 64 segments' at most, are joined in 64 bits. Each addition is off by
# 2^-24 of the sum, the exponential by 2^-23, its argument (log2 units of at most 4 above
# the reference, the weight of a lower one falls faster than its rounding grows) by 4 ln 2
# 2^-24: in all (16 + 128 + 6 + 2 + 3) 2^-24 of the sum, so of lse in absolute terms.
LSE = 155 * 2.0 ** -24


def candidates(x, scores, finished, eos):
    """[R, B V] in 64 bits, -inf where there is none."""
    R, B = scores.shape
    x = x.double().cpu().view(R, B, -1)
    s = scores.double().cpu()
    c = x - torch.logsumexp(x, -1, keepdim=True) + s[..., None]
    c[~torch.isfinite(x).all(-1) & (x.isnan() | (x == math.inf)).any(-1)] = -math.inf
    c[~(s > -math.inf)] = -math.inf
    if finished is not None:
        f = finished.cpu() & (s > -math.inf)
        c[f] = -math.inf
        c[..., eos] = torch.where(f, s, c[..., eos])
    c = torch.where(c.isnan(), -math.inf, c)
    return c.view(R, -1)


def check(x, scores, K=None, finished=None, eos=None, exact=False):
    """exact: beams' lse are alike or far apart, so the choice has to be the definition's."""
    R, B = scores.shape
    V = x.shape[1]
    K = K or B
    got = ops.beam_select(x, scores, K, finished, eos)
    c = candidates(x, scores, finished, eos)
    values, at = torch.sort(c, dim=-1, descending=True, stable=True)
    values, at = values[:, :K], at[:, :K]
    there = values > -math.inf
    s, p, t, f = (v.cpu() for v in got)
    assert s.shape == p.shape == t.shape == f.shape == (R, K)
    assert torch.equal(s > -math.inf, there)
    assert torch.equal(p[~there].long(), (B * torch.arange(R)[:, None]).expand(R, K)[~there])
    assert not t[~there].any() and not f[~there].any()
    flat = (p.long() - B * torch.arange(R)[:, None]) * V + t
    assert ((flat >= 0) & (flat < B * V)).all()
    for r in range(R):
        mine = flat[r][there[r]].tolist()
        assert len(set(mine)) == len(mine)
    bar = LSE + 2.0 ** -24 * values.abs()
    chosen = c.gather(1, flat)
    # the value it reports is the chosen candidate's, and that is the definition's, but
    # for candidates that lie closer together than the sums know
    assert ((s.double() - chosen).abs() <= bar)[there].all()
    assert ((chosen - values).abs() <= 2 * LSE)[there].all()
    alike = flat == at
    if exact:
        assert alike[there].all()
    else:
        gap = torch.full_like(values, math.inf)
        gap[:, 1:] = values[:, :-1] - values[:, 1:]
        nxt = torch.full_like(values, math.inf)
        nxt[:, :-1] = gap[:, 1:]
        clear = there & (gap > 2 * LSE) & (nxt > 2 * LSE)
        clear[:, -1] = False  # (the one behind the last may be close)
        assert alike[clear].all()
    want_f = torch.zeros_like(f)
    if eos is not None:
        want_f = t == eos
        if finished is not None:
            want_f |= finished.cpu().view(-1)[p.long()]
    assert torch.equal(f, want_f & there)
    return got


def logits(R, B, V, dt, seed, masked=0.0, spread=3.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = spread * torch.randn((R * B, V), generator=g, device=DEV)
    if masked:
        gone = torch.rand((R * B, V), generator=g, device=DEV) < masked
        gone[:, V // 2] = False
        x.masked_fill_(gone, -math.inf)
    return x.to(dt), -20 * torch.rand((R, B), generator=g, device=DEV)


@pytest.mark.parametrize("R,B,K,V,dt,masked", [
    (1, 1, 1, 1, BF, 0), (1, 1, 5, 7, F32, 0), (3, 2, 2, 1023, FP, 0.5), (2, 4, 8, 1024, BF, 0),
    (2, 4, 4, 1025, F32, 0.9), (1, 4, 4, 151936, BF, 0), (5, 3, 64, 4099, FP, 0.2),
    (2, 64, 64, 300, F32, 0), (1, 64, 64, 32001, BF, 0), (37, 5, 10, 65537, FP, 0.9),
    (128, 4, 4, 2050, BF, 0), (600, 1, 3, 1500, F32, 0), (300, 2, 4, 9000, BF, 0.99),
    (1, 2, 3, 1 << 20, F32, 0), (4096, 1, 1, 40, FP, 0), (70, 9, 20, 33, BF, 0.7),
])
def test_choice(R, B, K, V, dt, masked):
    x, s = logits(R, B, V, dt, R * 7 + V, masked)
    check(x, s, K)


@pytest.mark.parametrize("R,B,K,V", [(3, 5, 5, 777), (2, 8, 16, 20000), (200, 3, 3, 100)])
def test_finished_and_dead_beams(R, B, K, V):
    x, s = logits(R, B, V, BF, V)
    g = torch.Generator().manual_seed(V)
    f = (torch.rand((R, B), generator=g) < 0.4).to(DEV)
    s[0] = -math.inf       # nothing at all in the first prompt
    s[1, 1:] = -math.inf   # a first step: one beam
    f[1] = False
    s[-1, 0], f[-1] = -3.5, True  # all have ended
    x[f.view(-1)] = math.nan  # logits of ended beams are not read
    x[s.view(-1) == -math.inf] = math.nan
    got = check(x, s, K, f, V - 1)
    assert got.finished[-1, 0] and got.scores[-1, 0] == s[-1].max()
    check(x, s, K, f, 0)


def test_tokens_that_end():
    x, s = logits(2, 3, 50, F32, 5)
    x[:, 17] = 30.0
    got = check(x, s, 6, None, 17)
    assert got.finished[:, :3].all() and not got.finished[:, 3:].any()
    check(x, s, 6, torch.zeros((2, 3), dtype=torch.bool, device=DEV), 17)


@pytest.mark.parametrize("dt,V", [(BF, 4096), (FP, 4099), (F32, 1021), (BF, 151937)])
def test_ties(dt, V):
    """Beams of the same logits and scores: the lowest beam, then the lowest token,
    wherever their rows lie."""
    g = torch.Generator(device=DEV).manual_seed(V)
    row = torch.randint(-3, 4, (V,), generator=g, device=DEV).to(dt)
    x = row.expand(8, V).contiguous()
    check(x, torch.full((2, 4), -1.25, device=DEV), 16, exact=True)
    check(torch.zeros((6, V), dtype=dt, device=DEV), torch.zeros((2, 3), device=DEV), 64, exact=True)
    # a beam better by one step of fp32
    s = torch.tensor([[-1.0, math.nextafter(-1.0, 0.0), -1.0, -1.0]] * 2, device=DEV)
    s[:, 1] = -1.0 + 2.0 ** -24
    got = check(x, s, 3, exact=True)
    assert (got.parents == torch.tensor([[1], [5]], device=DEV)).all()


def test_values_that_are_not_finite():
    x, s = logits(3, 4, 3000, F32, 9)
    x[1, 5] = math.nan
    x[2, 2999] = math.inf
    x[3] = -math.inf
    x[4:8] = -math.inf    # a prompt without any candidate
    x[8:12, 1:] = -math.inf   # one a beam
    s[2, 3] = math.nan
    got = check(x, s, 8)
    assert (got.parents[0] == 0).all() and (got.scores[1] == -math.inf).all()
    assert (got.scores[2, 3:] == -math.inf).all()


@pytest.mark.parametrize("value", [-1e10, torch.finfo(F32).min, -65504.0, 1e30])
def test_large_finite_values(value):
    """Masks of finite values, whole rows of them, and rows of large ones."""
    x, s = logits(2, 3, 5000, F32, 11)
    x[:, ::2] = value
    x[4] = value
    # within a beam the order is the logits'; across beams such candidates tie in 64 bits
    check(x, s, 4)


def test_rows_of_a_wider_array_and_odd_addresses():
    x, s = logits(4, 3, 2049, BF, 13)
    want = ops.beam_select(x, s, 5)
    wide = torch.full((12, 2060), 50.0, dtype=BF, device=DEV)
    wide[:, 3:2052] = x
    for a, b in zip(ops.beam_select(wide[:, 3:2052], s, 5), want):
        assert torch.equal(a, b)
    t = x.t().contiguous().t()
    for a, b in zip(ops.beam_select(t, s, 5), want):
        assert torch.equal(a, b)
    one = x[:1].expand(6, 2049)  # rows of stride 0
    check(one, s[:2], 3, exact=True)


def test_rows_do_not_depend_on_their_neighbours():
    """A prompt's choice is the same alone and among many (split over workgroups
    another way: values to the sums' last bits)."""
    x, s = logits(130, 4, 5000, FP, 17)
    whole = ops.beam_select(x, s)
    for r in (0, 77, 129):
        alone = ops.beam_select(x[4 * r:4 * r + 4], s[r:r + 1])
        assert torch.equal(alone.tokens[0], whole.tokens[r])
        assert torch.equal(alone.parents[0] + 4 * r, whole.parents[r])
        assert ((alone.scores[0] - whole.scores[r]).abs() <= 2 * LSE + 2 ** -22 * 40).all()


def test_no_prompts():
    got = ops.beam_select(torch.zeros((0, 9), device=DEV), torch.zeros((0, 4), device=DEV), 2)
    assert got.tokens.shape == (0, 2)


def test_graph_and_streams():
    """Captured and replayed with other inputs and eager calls between; calls on two
    streams at once."""
    x, s = logits(6, 4, 30000, BF, 19)
    f = torch.zeros((6, 4), dtype=torch.bool, device=DEV)
    sx, ss, sf = x.clone(), s.clone(), f.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with hip.graph_workspaces(), torch.cuda.graph(graph):
        out = ops.beam_select(sx, ss, 4, sf, 3)
    for seed in range(4):
        x, s = logits(6, 4, 30000, BF, 23 + seed)
        f[:, seed] = True
        sx.copy_(x), ss.copy_(s), sf.copy_(f)
        graph.replay()
        want = ops.beam_select(x, s, 4, f, 3)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [ops.beam_select(x, s, 4, f, 3) for _ in range(20)]
    here = [ops.beam_select(x, s, 4, f, 3) for _ in range(20)]
    torch.cuda.synchronize()
    for r in there + here:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
