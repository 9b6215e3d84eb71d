"""Rows of attention behind shared prefixes whose scores are no numbers: NaN, as in the
paged attention, however the plan cut their keys."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from test_paged_gpu import BF, FP, gen_of, i32, rnd  # noqa: E402
from test_shared_gpu import make_cache  # noqa: E402

NAN = float("nan")


def step(R, H, HK, D, dtype, own=40, extra=()):
    """R single tokens behind 384 shared keys, then requests of `extra` keys by themselves."""
    g = gen_of(R + H + D)
    kv = [384 + 1 + (7 * r) % own for r in range(R)] + list(extra)
    kp, vp, table, *_ = make_cache(g, [(24, kv[:R])] + [(0, [n]) for n in extra], 16, HK, D, dtype)
    kp, vp = kp.nan_to_num(0.5), vp.nan_to_num(0.25)
    table = table.clamp(0, kp.shape[0] - 1)
    T = len(kv)
    cu, lens = i32(list(range(T + 1))), i32(kv)
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, R]), 16, T, H, HK, D)
    assert plan.keys.tolist() == [384]
    return rnd(g, T, H, D, dtype=dtype), kp, vp, table, cu, lens, plan


def both(q, kp, vp, table, cu, lens, plan, scale):
    got = ops.paged_shared_attention(q, kp, vp, table, plan, scale).isnan()
    want = ops.paged_attention(q, kp, vp, table, cu, lens, scale, 1).isnan()
    assert torch.equal(got, want)
    return got


# (rows joined by eight groups of lanes, and by one; a group of one narrow block, of one
# wide one, of several)
SIZES = [(4, 8, 2, 64, BF), (12, 8, 2, 128, FP), (48, 32, 8, 128, BF), (70, 16, 2, 64, FP)]


@pytest.mark.parametrize("R,H,HK,D,dtype", SIZES)
def test_in_one_row_of_q(R, H, HK, D, dtype):
    """In a request of the group, and in one cut in several parts by itself."""
    q, *rest = step(R, H, HK, D, dtype, extra=(6000, 500))
    q[R // 2, 3, 5] = q[R, 1, 0] = NAN
    got = both(q, *rest, D ** -0.5)
    want = torch.zeros_like(got)
    want[R // 2, 3] = want[R, 1] = True
    assert torch.equal(got, want)


@pytest.mark.parametrize("R,H,HK,D,dtype", SIZES)
def test_scale(R, H, HK, D, dtype):
    q, *rest = step(R, H, HK, D, dtype, extra=(6000, 5))
    assert both(q, *rest, NAN).all()


@pytest.mark.parametrize("R,H,HK,D,dtype", SIZES)
@pytest.mark.parametrize("where", ["prefix", "all of the prefix", "own", "alone"])
def test_in_the_keys_of_a_part(R, H, HK, D, dtype, where):
    """All keys of a part, and of several."""
    q, kp, vp, table, cu, lens, plan = step(R, H, HK, D, dtype, extra=(6000,))
    pages = {"prefix": table[0, 8:16], "all of the prefix": table[0, :24],
             "own": table[1, 24:25], "alone": table[R, 16:24]}[where].long()
    kp[pages, 0] = NAN
    rows = {"own": slice(1, 2), "alone": slice(R, R + 1)}.get(where, slice(0, R))
    if where == "own":  # (one key of its own or more, all on that page)
        assert int(lens[1]) <= 400
    got = both(q, kp, vp, table, cu, lens, plan, D ** -0.5)
    want = torch.zeros_like(got)
    want[rows, :H // HK] = True
    assert torch.equal(got, want)


def test_a_refused_request_beside_them():
    """No keys: zeros, whatever its group's prefix and q hold."""
    q, kp, vp, table, cu, lens, _ = step(12, 8, 2, 64, BF)
    kp[table[0, 3].long()] = NAN
    vp[table[0, 5].long()] = float("inf")
    q[5] = NAN
    lens[5] = 0
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, 12]), 16, 12, 8, 2, 64)
    got = ops.paged_shared_attention(q, kp, vp, table, plan, 0.125)
    assert plan.keys.tolist() == [384] and not got[5].any()
    rest = [r for r in range(12) if r != 5]
    assert got[rest].isnan().all()
