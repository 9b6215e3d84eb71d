"""How exactly beam selection's log sums are formed, over the longest rows."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402

DEV = "cuda"
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def check(x, bar):
    """Each row a prompt of one beam, whose score is such that the best candidate's lies
    near 0, where fp32 holds lse's error itself."""
    want, scores = [], []
    for row in x:  # (a row at a time: 64 bits of all would be large)
        d = row.double()
        best = d.max() - torch.logsumexp(d, 0)
        scores.append((-best).float())
        want.append(best + scores[-1].double())
    got = ops.beam_select(x, torch.stack(scores)[:, None], 1)
    err = (got.scores[:, 0].double() - torch.stack(want)).abs()
    assert float(err.max()) <= bar * U + U * float(torch.stack(want).abs().max()), float(err.max()) / U


@pytest.mark.parametrize("R", [8, 200])  # (rows over several workgroups, and in one)
@pytest.mark.parametrize("V,dt", [(1 << 20, BF), (151936, FP), ((1 << 20) - 3, F32), (1024, BF)])
def test_rows_of_one_value(R, V, dt):
    """All terms are alike, so every rounding of them or of their sums goes the same way.
    The exponential is off by one step, 2 x 2^-24, its argument, at most 1/2 and a fused
    product, by 2^-26 at most, as little again of the sum; sums of 16 equal terms in pairs
    and of chunks in 64 bits by nothing, the row's ragged end's by 4 x 2^-24 of a part of it
    (a 64th of 1024 values in the shortest row): 3 x 2^-24."""
    g = torch.Generator(device=DEV).manual_seed(V + R)
    values = (8 * torch.randn((R, 1), generator=g, device=DEV)).to(dt)
    check(values.expand(R, V), 3)


@pytest.mark.parametrize("R", [8, 200])
@pytest.mark.parametrize("V,dt", [(1 << 20, BF), (151936, FP), ((1 << 20) - 3, F32)])
def test_a_likely_token_over_a_tail(R, V, dt):
    """One value d above all others. Beside the exponential's 2 x 2^-24 and 4 for the sum
    of a chunk's 16 in pairs: an argument of t log2 units is rounded to |t| 2^-24 (half a
    step), of the sum's terms on average at most log2 V (a distribution's mean distance from
    its likeliest value is at most its entropy's bound, ln V) and 4 for the reference's
    place, times ln 2: 16.6 x 2^-24; what log2 e lacks in fp32, 1.34e-8 of that distance (in
    nats, 13.9): 3.2 x 2^-24. In all 26 x 2^-24."""
    g = torch.Generator(device=DEV).manual_seed(V + R)
    x = (4 * torch.randn((R, 1), generator=g, device=DEV)).to(dt).expand(R, V).contiguous()
    d = 2 + 14 * torch.rand(R, generator=g, device=DEV)
    x[torch.arange(R, device=DEV), torch.randint(0, V, (R,), generator=g, device=DEV)] += d.to(dt)
    check(x, 26)


@pytest.mark.parametrize("V,dt,spread", [(151936, BF, 3.0), (1 << 20, F32, 1.0), (65537, FP, 0.1)])
def test_random_rows(V, dt, spread):
    """The same bound, where the roundings differ."""
    g = torch.Generator(device=DEV).manual_seed(V)
    check((spread * torch.randn((24, V), generator=g, device=DEV)).to(dt), 26)
