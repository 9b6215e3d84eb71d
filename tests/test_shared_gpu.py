"""Attention behind shared prefixes against plain 64-bit attention of every request by
itself, and the shared keys against their definition."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import hip, ops  # noqa: E402

from test_paged_gpu import attention_64, check_attention, gen_of, i32, rnd  # noqa: E402

DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


def make_cache(g, groups, page, HK, D, dtype, extra=2):
    """groups: of each (shared pages, keys of each request); a request with fewer full
    pages has its own. What no key lies in is NaN. (k pool, v pool, table, keys and
    values of each request)."""
    pools, pages, rows, ks, vs = [], [], [], [], []
    total = sum(s + sum(-(-n // page) for n in kv) for s, kv in groups) + extra
    order = torch.randperm(total, generator=g).tolist()
    kp = torch.full((total, HK, page, D), float("nan"), dtype=dtype)
    vp = kp.clone()
    W = max([1] + [-(-n // page) for _, kv in groups for n in kv]) + 1

    def put(k, v):
        """Keys and values into new pages."""
        ids = []
        for a in range(0, k.shape[0], page):
            p = order.pop()
            m = min(page, k.shape[0] - a)
            kp[p, :, :m], vp[p, :, :m] = k[a:a + m].transpose(0, 1), v[a:a + m].transpose(0, 1)
            ids.append(p)
        return ids

    def rand(n):
        return tuple(torch.randn((n, HK, D), generator=g).to(dtype) for _ in range(2))

    for shared, kv in groups:
        pk, pv = rand(shared * page)
        prefix = put(pk, pv)
        for n in kv:
            m = shared if n >= shared * page else 0
            k, v = rand(n - m * page)
            ids = prefix[:m] + put(k, v)
            rows.append(ids + [-1, total + 3, 2 ** 31 - 1] * W)
            ks.append(torch.cat([pk[:m * page], k]))
            vs.append(torch.cat([pv[:m * page], v]))
    table = [r[:W] for r in rows]
    return kp.to(DEV), vp.to(DEV), i32(table), ks, vs


def shared_by_hand(table, kv, n_q, groups, page):
    out = []
    for a, b in zip(groups, groups[1:]):
        some = [r for r in range(a, b) if n_q[r] and kv[r] > 0]
        n = 0
        if some:
            most = min(max(kv[r] - n_q[r], 0) // page for r in some)
            while n < most and len({table[r][n] for r in some}) == 1:
                n += 1
        out.append(n * page)
    return out


def run(groups, n_q, H, HK, D, page, dtype, cu_groups=None, seed=0, scale=None, spare=0):
    g = gen_of(seed + D + page + len(n_q))
    kp, vp, table, ks, vs = make_cache(g, groups, page, HK, D, dtype)
    kv = [n for _, lens in groups for n in lens]
    if cu_groups is None:
        cu_groups = np.cumsum([0] + [len(lens) for _, lens in groups]).tolist()
    T = sum(n_q)
    q = rnd(g, T + spare, H, D, dtype=dtype)
    cu, lens = i32([0] + np.cumsum(n_q).tolist()), i32(kv)
    scale = D ** -0.5 if scale is None else scale
    plan = ops.paged_shared_plan(table, cu, lens, i32(cu_groups), page, T + spare, H, HK, D)
    assert plan.keys.tolist() == shared_by_hand(table.tolist(), kv, n_q, cu_groups, page)
    out = ops.paged_shared_attention(q, kp, vp, table, plan, scale)
    check_attention(out[:T], *attention_64(q[:T], ks, vs, n_q, scale), dtype)
    return out, plan, (q, kp, vp, table, cu, lens, scale)


@pytest.mark.parametrize("groups,n_q,H,HK,D,page,dtype", [
    ([(1, [17])], [1], 8, 2, 64, 16, BF),                                # one request
    ([(0, [1, 2])], [1, 1], 8, 2, 128, 16, FP),                          # nothing shared
    ([(15, [1000, 977, 961, 1010])], [1] * 4, 32, 8, 128, 64, BF),       # beams
    ([(7, [130, 113, 120])], [1] * 3, 8, 2, 64, 16, BF),                 # 112 keys: not worth it
    ([(8, [130, 129, 150])], [1] * 3, 8, 2, 128, 16, BF),                # 128
    ([(9, [145, 146, 400])], [1] * 3, 8, 2, 64, 16, FP),                 # 144: half a tile over
    ([(2, [257, 300, 512, 259])], [1] * 4, 4, 1, 128, 128, BF),
    ([(4, [1025, 1500, 2000])], [1] * 3, 16, 2, 64, 256, BF),            # 24 columns
    ([(20, [640 + i for i in range(1, 10)])], [1] * 9, 32, 8, 128, 32, FP),   # 36 columns: wide
    ([(20, [640 + 9 * i for i in range(1, 34)])], [1] * 33, 32, 8, 64, 32, BF),   # 132: two blocks
    ([(30, [500 + i for i in range(64)])], [1] * 64, 40, 8, 128, 16, BF),   # 5 q heads a kv head
    ([(10, [700, 650, 900])], [4, 1, 7], 16, 2, 64, 64, FP),             # a few tokens each
    ([(40, [700, 650, 900, 641])], [16, 2, 9, 1], 8, 2, 128, 16, BF),    # 64 columns a request
    ([(40, [700, 650, 900, 641])], [17, 2, 9, 1], 8, 2, 128, 16, BF),    # 68: by themselves
    ([(12, [200, 400]), (0, [33]), (5, [700, 90, 650]), (30, [500, 600])],
     [1, 2, 33, 1, 5, 1, 1, 3], 8, 2, 64, 16, BF),
    ([(12, [300, 0, 250, 400]), (9, [0, 0])], [1, 1, 0, 2, 0, 1], 8, 2, 128, 16, FP),
    ([(3, [200, 192, 193]), (3, [300, 7])], [8, 1, 1, 1, 2], 8, 1, 128, 64, BF),   # its step's own keys
    ([(2, [128, 129]), (2, [3, 600])], [128, 1, 5, 3], 4, 2, 64, 64, BF),
    ([(100, [6500] * 4 + [9000, 6401])], [1] * 6, 32, 8, 64, 64, FP),
    ([(600, [9700, 9650, 9601])], [1, 2, 1], 32, 4, 128, 16, BF),
    ([(1, [600]), (1, [300]), (1, [2000])], [600, 150, 1], 8, 2, 128, 32, BF),     # prompts
    ([(3, [50, 60])], [1, 1], 40, 1, 64, 16, BF),
    ([(16, [300, 290, 280])], [1] * 3, 128, 1, 64, 16, FP),              # 128 columns a request
])
def test_attention(groups, n_q, H, HK, D, page, dtype):
    run(groups, n_q, H, HK, D, page, dtype)


@pytest.mark.parametrize("seed", range(6))
def test_random_batches(seed):
    rng = np.random.default_rng(200 + seed)
    page, D = [16, 32, 64, 16, 128, 256][seed], [64, 128][seed % 2]
    groups, n_q = [], []
    for _ in range(int(rng.integers(1, 12))):
        shared = int(rng.choice([0, 1, 3, 128 // page + 1, 700 // page + 1]))
        kv = [int(shared * page + rng.choice([0, 1, 5, 130, 400]) + rng.integers(0, 3))
              for _ in range(int(rng.integers(1, 14)))]
        few = int(rng.choice([1, 1, 3, 9, 40]))
        groups.append((shared, kv))
        n_q += [int(min(rng.integers(0, few + 1), n)) if rng.random() < 0.9 else 0 for n in kv]
    n_q[0] = max(n_q[0], 1)
    G, HK = [(4, 2), (8, 1), (1, 4), (5, 2), (2, 2), (16, 1)][seed]
    run(groups, n_q, G * HK, HK, D, page, [BF, FP][seed % 2], seed=seed)


@pytest.mark.parametrize("R", [65, 300, 2500])
def test_many_requests(R):
    rng = np.random.default_rng(R)
    groups, n_q = [], []
    while len(n_q) < R:
        n = min(int(rng.integers(1, 40)), R - len(n_q))
        shared = int(rng.integers(0, 20)) if rng.random() < 0.3 else 0
        groups.append((shared, (16 * shared + rng.integers(1, 30, n)).tolist()))
        n_q += np.minimum(rng.integers(0, 3, n), 1).tolist()
    n_q[-1] = 1
    run(groups, n_q, 4, 2, 64, 16, BF)


def test_groups_that_leave_requests_out():
    """Requests before, behind and between groups, empty groups, groups of one."""
    groups = [(12, [300, 250, 260, 400, 210, 200])]
    for cu in ([0, 6], [2, 5], [0, 0, 1, 4, 4], [1, 3, 6, 6], [5, 5], [0, 1, 2, 3, 4, 5, 6]):
        run(groups, [1, 1, 2, 1, 1, 1], 8, 2, 64, 16, BF, cu_groups=cu)


def test_rows_behind_the_last_request():
    out, plan, (q, kp, vp, table, cu, lens, scale) = run([(12, [300, 250])], [1, 2], 8, 2, 128, 16, BF,
                                                         spare=5)
    mark = torch.full_like(q, 7.0)
    hip.paged_shared_attention(q, kp, vp, mark, table, plan, scale)
    assert (mark[3:] == 7.0).all() and torch.equal(mark[:3], out[:3])


@pytest.mark.parametrize("scale", [-0.09, 0.0])
def test_scales(scale):
    run([(12, [300, 250, 260, 400] * 3)], [1] * 12, 8, 2, 128, 16, BF, scale=scale)


def test_large_scores():
    """Scores that differ by hundreds, of both signs, between prefix and rest."""
    run([(12, [300, 250, 260, 400] * 3)], [1] * 12, 8, 2, 64, 16, FP, scale=8.0)


def test_beside_values_that_are_not_finite():
    """In one request's own keys: no other request knows. In the prefix: all of its
    group know, no other."""
    kv = [300, 250, 400]
    g = gen_of(71)
    kp, vp, table, ks, vs = make_cache(g, [(12, kv), (12, kv)], 16, 2, 64, BF)
    q, cu, lens = rnd(g, 6, 8, 64), i32(list(range(7))), i32(kv * 2)
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, 3, 6]), 16, 6, 8, 2, 64)
    assert plan.keys.tolist() == [192, 192]
    want, size = attention_64(q, ks, vs, [1] * 6, 0.125)
    for bad in (float("nan"), float("inf")):
        k, v = kp.clone(), vp.clone()
        k[table[1, 249 // 16], :, 249 % 16] = bad
        v[table[1, 249 // 16], :, 249 % 16] = bad
        out = ops.paged_shared_attention(q, k, v, table, plan, 0.125)
        keep = [0, 2, 3, 4, 5]
        check_attention(out[keep], want[keep], size[keep], BF)
        assert not out[1].isfinite().any()
        k, v = kp.clone(), vp.clone()
        v[table[0, 3], :, 5] = bad
        out = ops.paged_shared_attention(q, k, v, table, plan, 0.125)
        check_attention(out[3:], want[3:], size[3:], BF)
        assert (out[:3] == bad).all() if bad == float("inf") else out[:3].isnan().all()


def test_a_refused_request_in_a_group():
    """A request whose step was refused (no keys) has tokens among its group's."""
    groups, n_q = [(12, [300, 250, 260, 280] * 4)], [1] * 16
    out, plan, (q, kp, vp, table, cu, lens, scale) = run(groups, n_q, 8, 2, 64, 16, BF)
    lens[5] = 0
    again = ops.paged_shared_plan(table, cu, lens, i32([0, 16]), 16, 16, 8, 2, 64, out=plan)
    got = ops.paged_shared_attention(q, kp, vp, table, again, scale)
    assert not got[5].any() and plan.keys.tolist() == [192]
    rest = [i for i in range(16) if i != 5]
    assert float((got[rest].float() - out[rest].float()).abs().max()) < 0.02


def test_a_refused_prompt_in_a_group():
    """One whose step was refused has a thousand tokens among single ones."""
    g = gen_of(73)
    kv, n_q = [300, 0, 260, 280, 250], [1, 1000, 1, 1, 2]
    kp, vp, table, ks, vs = make_cache(g, [(12, kv)], 16, 2, 64, BF)
    T = sum(n_q)
    q, cu, lens = rnd(g, T, 8, 64), i32([0] + np.cumsum(n_q).tolist()), i32(kv)
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, 5]), 16, T, 8, 2, 64)
    assert plan.keys.tolist() == [192] and int(plan.schedule[0]) > 0
    out = ops.paged_shared_attention(q, kp, vp, table, plan, 0.125)
    check_attention(out, *attention_64(q, ks, vs, n_q, 0.125), BF)
    assert not out[1:1001].any()


def test_offsets_that_fall():
    """Nothing is written where they do, and the next plan is as before."""
    out, plan, (q, kp, vp, table, cu, lens, scale) = run([(12, [300, 250, 260])], [1, 2, 1], 8, 2, 64, 16,
                                                         BF)
    sizes = (16, 4, 8, 2, 64)
    for bad_cu, bad_groups in ((i32([0, 3, 1, 4]), i32([0, 3])), (cu, i32([3, 0]))):
        again = ops.paged_shared_plan(table, bad_cu, lens, bad_groups, *sizes, out=plan)
        mark = torch.full_like(q, 7.0)
        hip.paged_shared_attention(q, kp, vp, mark, table, again, scale)
        assert (mark == 7.0).all()
    ops.paged_shared_plan(table, cu, lens, i32([0, 3]), *sizes, out=plan)
    assert torch.equal(ops.paged_shared_attention(q, kp, vp, table, plan, scale), out)


def test_a_plan_of_other_sizes():
    """The C entry with a schedule made for other sizes: out stays as it was."""
    out, plan, (q, kp, vp, table, cu, lens, scale) = run([(12, [300, 250, 260])], [1, 2, 1], 8, 2, 64, 16,
                                                         BF)
    big = torch.zeros(1 << 20, dtype=torch.int32, device=DEV)
    big[:plan.schedule.numel()] = plan.schedule
    other = ops.SharedPlan(plan.keys, big, (3,) + plan.shape[1:])
    mark = torch.full_like(q, 7.0)
    hip.paged_shared_attention(q[:3], kp, vp, mark, table, other, scale)
    assert (mark == 7.0).all()


def test_no_tokens():
    table, i = i32([[0, 0], [0, 0]]), i32([0, 0])
    plan = ops.paged_shared_plan(table, i32([0, 0, 0]), i, i32([0, 2]), 16, 0, 4, 2, 64)
    pool = torch.zeros((2, 2, 16, 64), dtype=BF, device=DEV)
    out = ops.paged_shared_attention(torch.zeros((0, 4, 64), dtype=BF, device=DEV), pool, pool, table,
                                     plan, 1.0)
    assert plan.keys.tolist() == [0] and out.shape == (0, 4, 64)


def test_strides_and_alignment_of_q():
    out, plan, (q, kp, vp, table, cu, lens, scale) = run([(12, [300, 250] * 4)], [1] * 8, 8, 2, 64, 16, BF)
    wide = torch.full((8, 8, 72), 9.0, dtype=BF, device=DEV)
    wide[..., 3:67] = q
    assert torch.equal(ops.paged_shared_attention(wide[..., 3:67], kp, vp, table, plan, scale), out)
    t = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ops.paged_shared_attention(t, kp, vp, table, plan, scale), out)


def test_a_long_prefix_in_a_large_pool():
    """Offsets past 32 bits in the pools, 70001 keys in all."""
    page, HK, D, P = 256, 8, 128, 9000  # 4.7 GB a pool
    g = torch.Generator(device=DEV).manual_seed(3)
    pools = [torch.empty((P, HK, page, D), dtype=BF, device=DEV).normal_(generator=g) for _ in range(2)]
    order = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    order[:2] = torch.tensor([P - 1, P - 2], device=DEV)
    table = torch.empty((5, 280), dtype=torch.int32, device=DEV)
    table[:, :270] = order[:270]
    table[:, 270:] = order[300:350].view(5, 10)
    lens = i32([70001, 69200, 69121, 70100, 70900])
    q = torch.empty((5, 32, D), dtype=BF, device=DEV).normal_(generator=g)
    cu = i32(list(range(6)))
    plan = ops.paged_shared_plan(table, cu, lens, i32([0, 5]), page, 5, 32, HK, D)
    assert plan.keys.tolist() == [270 * page]
    got = ops.paged_shared_attention(q, *pools, table, plan, D ** -0.5)
    ks, vs = ([p[table[r].long()].transpose(1, 2).reshape(-1, HK, D)[:n].cpu()
               for r, n in enumerate(lens.tolist())] for p in pools)
    check_attention(got, *attention_64(q, ks, vs, [1] * 5, D ** -0.5), BF)


def test_graph_of_plan_and_layers():
    """A step's plan and two layers' attention captured, replayed at other lengths and
    tables with eager work between."""
    g = gen_of(41)
    groups = [(12, [300, 250, 260, 400]), (20, [330, 400, 500])]
    kp, vp, table, *_ = make_cache(g, groups, 16, 2, 64, BF)
    kp, vp = kp.nan_to_num(0.5), vp.nan_to_num(0.25)
    table = table.clamp(0, kp.shape[0] - 1)
    lens, cu = i32([n for _, kv in groups for n in kv]), i32(list(range(8)))
    gr = i32([0, 4, 7])
    q = [rnd(g, 7, 8, 64) for _ in range(2)]

    def step(plan=None):
        p = ops.paged_shared_plan(table, cu, lens, gr, 16, 7, 8, 2, 64, out=plan)
        return p, [ops.paged_shared_attention(x, kp, vp, table, p, 0.125) for x in q]

    graph = torch.cuda.CUDAGraph()
    step()
    torch.cuda.synchronize()
    with hip.graph_workspaces(), torch.cuda.graph(graph):
        plan, outs = step()
    for i in range(5):
        lens += i32([1, 0, 2, 1, 0, 1, 3])
        lens[i] = 200 + i
        table[5 + i % 2, 3 * i:] = table[4, 3 * i:]
        graph.replay()
        p, want = step()
        assert torch.equal(p.keys, plan.keys), i
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_two_streams_and_repeats():
    out, plan, (q, kp, vp, table, cu, lens, scale) = run([(40, [700 + i for i in range(40)])], [1] * 40, 32,
                                                         8, 128, 16, BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [ops.paged_shared_attention(q, kp, vp, table, plan, scale) for _ in range(20)]
    here = [ops.paged_shared_attention(q, kp, vp, table, plan, scale) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) for x in there + here)
