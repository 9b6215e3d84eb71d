"""What the rounding of single tokens' attention probabilities leaves in the result."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from test_paged_gpu import BF, FP, gen_of, half_step, i32  # noqa: E402


@pytest.mark.parametrize("L,n,D,dtype", [(2, 1, 128, BF), (2, 1, 64, FP), (33, 1, 64, BF),
                                         (33, 1, 128, FP), (34, 5, 128, BF), (34, 8, 64, FP)])
def test_values_that_cancel(L, n, D, dtype):
    """Values of 1 and -1 in turn behind nearly equal scores: a result near 0, which a
    probability's error of half a step of its type (2^-9 in bf16, 2^-12 in fp16) passes
    by far. Held to half a step of the result; beside it a probability in two pieces is
    off by at most 2^-18 of itself, its exponential by 2^-22, sums of 34 terms by
    34 x 2^-24: under 2^-17 in all."""
    R, HK, page = 40, 2, 16
    g = gen_of(L + n)
    W = -(-L // page)
    k = torch.zeros((R, L, HK, D))
    k[..., 0] = -torch.rand((R, L, HK), generator=g) / 50
    v = torch.ones((R, L, HK, D))
    v[:, 1::2] = -1
    q = torch.zeros((R * n, 4 * HK, D))
    q[..., 0] = 1 + torch.rand((R * n, 4 * HK), generator=g)
    k, v, q = (t.to(dtype) for t in (k, v, q))

    def pool(x):
        full = torch.zeros((R, W * page, HK, D), dtype=dtype)
        full[:, :L] = x
        return full.view(R * W, page, HK, D).transpose(1, 2).contiguous().cuda()

    out = ops.paged_attention(q.cuda(), pool(k), pool(v), i32([[r * W + w for w in range(W)] for r in range(R)]),
                              i32([r * n for r in range(R + 1)]), i32([L] * R), 1.0, n)
    s = torch.einsum("rihd,rjhd->rihj", q.double().view(R, n, 4 * HK, D),
                     k.double().repeat_interleave(4, 2))
    s.masked_fill_(torch.arange(L)[None, None, None] > torch.arange(n)[None, :, None, None] + L - n, -1e300)
    want = torch.einsum("rihj,rjhd->rihd", torch.softmax(s, -1), v.double().repeat_interleave(4, 2))
    err = (out.double().cpu().view_as(want) - want).abs()
    assert bool((err <= half_step(dtype) * want.abs() + 2.0 ** -17).all()), float(err.max())


@pytest.mark.parametrize("L,D,dtype", [(3, 64, BF), (33, 128, BF), (700, 64, FP), (5000, 128, BF)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinite_values(L, D, dtype, bad):
    """A visible value that is infinite makes its column infinite, one that is no
    number no number; the other columns and the other request are what they are
    without it."""
    g = gen_of(L)
    page, HK = 32, 2
    W = -(-L // page)
    kp, vp = (torch.randn((2 * W, HK, page, D), generator=g).to(dtype).cuda() for _ in range(2))
    q = torch.randn((2, 8, D), generator=g).to(dtype).cuda()
    table = i32([list(range(W)), list(range(W, 2 * W))])
    args = (table, i32([0, 1, 2]), i32([L, L]), D ** -0.5, 1)
    want = ops.paged_attention(q, kp, vp, *args)
    j = L // 2
    vp[j // page, 1, j % page, 5] = bad
    got = ops.paged_attention(q, kp, vp, *args)
    column = got[0, 4:, 5].float()
    assert bool((column == bad).all()) if bad == bad else bool(column.isnan().all())
    got[0, 4:, 5] = want[0, 4:, 5]
    # (without the rests of the probabilities: half a step of each, at most 2^-8 of the
    # values' mean size, and half a step of the results)
    assert torch.equal(got[1], want[1]) and torch.equal(got[0, :4], want[0, :4])
    err = (got[0, 4:].double() - want[0, 4:].double()).abs()
    assert bool((err <= half_step(dtype) * (1 + 2 * want[0, 4:].double().abs())).all()), float(err.max())
