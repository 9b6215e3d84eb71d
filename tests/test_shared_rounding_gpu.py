"""What the rounding of the probabilities leaves in attention behind shared prefixes: no
more than in the paged attention, however many requests share."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from test_paged_gpu import BF, FP, attention_64, gen_of, half_step, i32, rnd  # noqa: E402
from test_shared_gpu import make_cache  # noqa: E402


@pytest.mark.parametrize("R,few,H,HK,D,page,dtype", [
    (33, 1, 8, 2, 128, 64, BF), (64, 1, 8, 2, 64, 16, FP), (96, 1, 4, 1, 128, 64, BF),
    (96, 4, 4, 1, 64, 64, FP), (40, 8, 4, 1, 128, 32, BF), (9, 1, 32, 2, 64, 16, BF),
    (5, 1, 32, 1, 128, 16, FP), (12, 3, 40, 4, 64, 64, BF),
])
def test_large_groups_round_once(R, few, H, HK, D, page, dtype):
    """Groups of more than 128 columns (a request's: at most 32) behind 1024 keys. A
    probability in two pieces is off by 2^-17 of itself at most (bf16), its exponential by
    2^-23, its score, 128 products whose sum is rounded at each, up or down, to 2^-24 of at
    most about 10 log2 units, by 5e-6: the result before its own rounding by less than 3e-5
    of its norm. Rounded, the definition's is off by 1.5e-3 of its norm in bf16 and 1.9e-4 in
    fp16; rounded probabilities leave as much again."""
    rng = np.random.default_rng(R + few)
    shared = 1024 // page
    n_q = rng.integers(1, few + 1, R).tolist()
    n_q[0] = few
    kv = [shared * page + n + int(rng.integers(0, 40)) for n in n_q]
    g = gen_of(R + D)
    kp, vp, table, ks, vs = make_cache(g, [(shared, kv)], page, HK, D, dtype)
    T = sum(n_q)
    assert T * H // HK > 128 and few * H // HK <= 32
    q, cu, lens = rnd(g, T, H, D, dtype=dtype), i32([0] + np.cumsum(n_q).tolist()), i32(kv)
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, R]), page, T, H, HK, D)
    assert plan.keys.tolist() == [1024]
    out = ops.paged_shared_attention(q, kp, vp, table, plan, D ** -0.5).double().cpu()
    want, _ = attention_64(q, ks, vs, n_q, D ** -0.5)
    rounding = (want.to(dtype).double() - want).norm()
    assert float((out - want).norm()) <= float(rounding) + 3e-5 * float(want.norm())


@pytest.mark.parametrize("n_q,H,HK,D,page,dtype", [
    ([40] * 6, 8, 2, 128, 64, BF), ([40, 9, 33, 1], 4, 4, 64, 16, FP), ([40, 40, 21], 16, 2, 64, 32, FP),
    ([128, 100], 8, 2, 128, 16, BF), ([17, 16, 20], 16, 4, 64, 64, BF), ([512], 2, 2, 128, 128, FP),
])
def test_steps_of_some_tokens_round_once(n_q, H, HK, D, page, dtype):
    """Requests by themselves of up to 512 columns: the bound above."""
    assert max(n_q) * H // HK <= 512
    R, T = len(n_q), sum(n_q)
    kv = [1200 + 37 * r for r in range(R)]
    g = gen_of(T + D)
    kp, vp, table, ks, vs = make_cache(g, [(0, kv)], page, HK, D, dtype)
    q, cu, lens = rnd(g, T, H, D, dtype=dtype), i32([0] + np.cumsum(n_q).tolist()), i32(kv)
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, R]), page, T, H, HK, D)
    out = ops.paged_shared_attention(q, kp, vp, table, plan, D ** -0.5).double().cpu()
    want, _ = attention_64(q, ks, vs, n_q, D ** -0.5)
    rounding = (want.to(dtype).double() - want).norm()
    assert float((out - want).norm()) <= float(rounding) + 3e-5 * float(want.norm())


@pytest.mark.parametrize("R,n,D,dtype", [(40, 1, 128, BF), (40, 1, 64, FP), (20, 8, 128, FP),
                                         (20, 8, 64, BF), (5, 1, 64, BF)])
def test_values_that_cancel(R, n, D, dtype):
    """Values of 1 and -1 in turn behind nearly equal scores, 160 of the keys shared: a
    result near 0, which a probability's error of half a step of its type passes by far.
    Held to half a step of the result; beside it a probability in two pieces is off by
    2^-18 of itself, its exponential by 2^-22, sums of 200 terms by 200 x 2^-24 (a value's
    terms are added by fours of 16, in fact): under 2^-15 in all."""
    HK, G, page, S, L = 2, 4, 16, 160, 200
    g = gen_of(R + n + D)
    own = -(-(L - S) // page)
    k = torch.zeros((R, L, HK, D))
    k[..., 0] = -torch.rand((R, L, HK), generator=g) / 50
    k[:, :S] = k[:1, :S]
    v = torch.ones((R, L, HK, D))
    v[:, 1::2] = -1
    q = torch.zeros((R * n, G * HK, D))
    q[..., 0] = 1 + torch.rand((R * n, G * HK), generator=g)
    k, v, q = (t.to(dtype) for t in (k, v, q))

    def pool(x):
        """The prefix's pages, then every request's own."""
        rest = torch.zeros((R, own * page, HK, D), dtype=dtype)
        rest[:, :L - S] = x[:, S:]
        both = torch.cat([x[0, :S].reshape(-1, page, HK, D), rest.reshape(-1, page, HK, D)])
        return both.transpose(1, 2).contiguous().cuda()

    first = S // page
    table = i32([[*range(first), *range(first + r * own, first + (r + 1) * own)] for r in range(R)])
    cu, lens = i32([r * n for r in range(R + 1)]), i32([L] * R)
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, R]), page, R * n, G * HK, HK, D)
    assert plan.keys.tolist() == [S]
    out = ops.paged_shared_attention(q.cuda(), pool(k), pool(v), table, plan, 1.0)
    want, _ = attention_64(q, list(k), list(v), [n] * R, 1.0)
    err = (out.double().cpu() - want).abs()
    assert bool((err <= half_step(dtype) * want.abs() + 2.0 ** -15).all()), float(err.max())
