"""Forking and compacting pages against their definitions, request after request."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import hip, ops  # noqa: E402

DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def pages_of(n, page, W):
    return min(-(-max(n, 0) // page), W)


def fork_by_hand(table, lens, sources, free, count, page, pools):
    """(table, lens, free, count, refused, pools), the arrays of the call as lists and
    the pools as numpy arrays."""
    R, W, P = len(table), len(table[0]), pools[0].shape[0]
    live = [pages_of(n, page, W) for n in lens]
    held = [min(max(n, 0), W * page) for n in lens]
    before = {p for r in range(R) for p in table[r][:live[r]]}
    after = {p for s in sources if 0 <= s < R for p in table[s][:live[s]]}
    gone = sorted(p for p in before - after if 0 <= p < P)
    stack = free[:count] + gone
    copies = []
    for s in range(R):
        heirs = [r for r in range(R) if sources[r] == s]
        if heirs and held[s] % page:
            copies += [r for r in heirs if r != (s if s in heirs else heirs[0])]
    refused = max(0, len(copies) - len(stack)) + sum(s >= R for s in sources)
    if refused:
        return table, lens, free, count, refused, pools
    new, pools = [list(r) for r in table], [p.copy() for p in pools]
    for r, s in enumerate(sources):
        if s >= 0:
            new[r][:live[s]] = table[s][:live[s]]
    pushed = stack + free[len(stack):]
    for j, r in enumerate(sorted(copies)):
        s = sources[r]
        old, page_id, rows = table[s][live[s] - 1], stack[len(stack) - 1 - j], held[s] % page
        new[r][live[s] - 1] = page_id
        for p in pools:
            p[page_id, :, :rows] = p[old, :, :rows]
    return (new, [lens[s] if s >= 0 else 0 for s in sources], pushed, len(stack) - len(copies), 0,
            pools)


def compact_by_hand(table, lens, free, count, page, pools):
    R, W, P = len(table), len(table[0]), pools[0].shape[0]
    live = [pages_of(n, page, W) for n in lens]
    used = sorted({p for r in range(R) for p in table[r][:live[r]] if 0 <= p < P})
    n = len(used)
    to = dict(zip([p for p in used if p >= n], sorted(set(range(n)) - set(used))))
    new, pools = [list(r) for r in table], [p.copy() for p in pools]
    for r in range(R):
        new[r][:live[r]] = [to.get(p, p) for p in table[r][:live[r]]]
    for a, b in to.items():
        for p in pools:
            p[b] = p[a]
    return new, list(range(P - 1, n - 1, -1)) + free[P - n:], P - n, n, pools


def batch(rng, R, page, kv, spare, share=0, W=None):
    """Requests of kv keys over a pool with `spare` free pages; the first `share` pages of
    request 0 are those of all that have as many full ones."""
    W = W or max(1, max(-(-n // page) for n in kv))
    live = [pages_of(n, page, W) for n in kv]
    ids = rng.permutation(sum(live) + spare).tolist()
    P = max(1, len(ids))
    table = [[ids.pop() if w < live[r] else -9 for w in range(W)] for r in range(R)]
    for r in range(1, R):
        if share and kv[r] // page >= share and kv[0] // page >= share:
            ids += table[r][:share]
            table[r][:share] = table[0][:share]
    return table, ids, P


def pools_of(rng, n, P, HK, page, D, dt):
    host = [rng.standard_normal((P, HK, page, D)).astype(np.float32) for _ in range(n)]
    dev = [torch.from_numpy(h).to(DEV).to(dt) for h in host]
    return [d.float().cpu().numpy() for d in dev], dev


def same_pools(dev, want):
    for d, w in zip(dev, want):
        assert np.array_equal(d.float().cpu().numpy(), w)


def run_fork(table, lens, sources, free, page, host, dev, extra=0):
    P = host[0].shape[0]
    padded = free + [-5] * (P + extra - len(free))
    want = fork_by_hand(table, lens, sources, padded, len(free), page, host)
    t, n, f, c = i32(table), i32(lens), i32(padded), i32([len(free)])
    refused = ops.paged_fork(t, n, i32(sources), f, c, ops.page_pools(dev))
    assert int(refused) == want[4]
    assert n.tolist() == want[1] and t.tolist() == want[0]
    assert int(c) == want[3] and f.tolist() == want[2]
    same_pools(dev, want[5])
    return t, n, f, c, want


@pytest.mark.parametrize("R,page,hi,share,HK,D,layers,dt,spare", [
    (1, 16, 40, 0, 1, 64, 1, BF, 2), (2, 16, 1, 0, 2, 64, 1, FP, 3), (4, 64, 700, 5, 8, 128, 3, BF, 6),
    (64, 16, 90, 2, 2, 64, 2, FP, 80), (65, 32, 300, 1, 1, 128, 1, BF, 70), (300, 256, 900, 1, 1, 64, 1,
    BF, 400), (1100, 16, 33, 0, 1, 64, 1, FP, 1200), (5, 128, 128, 0, 3, 128, 2, BF, 6),
    (4096, 16, 20, 0, 1, 64, 1, BF, 4100),
])
def test_fork(R, page, hi, share, HK, D, layers, dt, spare):
    """Some requests of length 0 and of whole pages; some end, some go on, some are
    replaced; then the same sources again."""
    rng = np.random.default_rng(R * 31 + page)
    kv = rng.integers(0, hi + 1, R).tolist()
    kv[0] = hi
    kv[-1] = kv[-1] // page * page
    table, free, P = batch(rng, R, page, kv, spare, share)
    sources = [int(s) if a < 0.5 else (r if a < 0.9 else -1) for r, (s, a) in
               enumerate(zip(rng.integers(0, R, R), rng.random(R)))]
    host, dev = pools_of(rng, 2 * layers, P, HK, page, D, dt)
    t, n, f, c, want = run_fork(table, kv, sources, free, page, host, dev, 3)
    run_fork(t.tolist(), n.tolist(), sources, f.tolist()[:int(c)], page, want[5], dev)


def test_fork_of_one_prompt_and_ends():
    """Samples of one prompt, then all but one end, then the last."""
    rng = np.random.default_rng(3)
    table, free, P = batch(rng, 8, 16, [37] + [0] * 7, 9)
    host, dev = pools_of(rng, 2, P, 2, 16, 64, BF)
    t, n, f, c, want = run_fork(table, [37] + [0] * 7, [0] * 8, free, 16, host, dev)
    assert n.tolist() == [37] * 8 and int(c) == len(free) - 7
    assert len(set(t[:, 2].tolist())) == 8 and len(set(t[:, 1].tolist())) == 1
    t, n, f, c, want = run_fork(t.tolist(), n.tolist(), [-1] * 5 + [6, -1, -1], f.tolist()[:int(c)],
                                16, want[5], dev)
    assert int(c) == P - 3 and n.tolist() == [0] * 5 + [37, 0, 0]
    t, n, f, c, want = run_fork(t.tolist(), n.tolist(), [-1] * 8, f.tolist()[:int(c)], 16, want[5], dev)
    assert int(c) == P and sorted(f.tolist()[:P]) == list(range(P))


def test_pages_that_run_out():
    """Three copies with two pages: nothing changes. With one that the fork itself sets
    free they reach."""
    rng = np.random.default_rng(5)
    kv = [20, 20, 20, 20]
    table, free, P = batch(rng, 4, 16, kv, 2)
    host, dev = pools_of(rng, 2, P, 1, 16, 64, BF)
    run_fork(table, kv, [0, 1, 2, 3], [], 16, host, dev)  # nothing to do: no page needed
    *_, want = run_fork(table, kv, [0, 0, 0, 0], [], 16, host, dev)  # six pages come back
    assert want[4] == 0
    host, dev = pools_of(rng, 2, P, 1, 16, 64, BF)
    *_, want = run_fork(table, [20, 0, 0, 0], [0, 0, 0, 0], free[:2], 16, host, dev)
    assert want[4] == 1
    *_, want = run_fork(table, [20, 5, 0, 0], [0, 0, 0, 0], free[:2], 16, host, dev)
    assert want[4] == 0


def test_sources_that_are_no_requests():
    rng = np.random.default_rng(7)
    table, free, P = batch(rng, 3, 16, [20, 40, 10], 4)
    host, dev = pools_of(rng, 1, P, 1, 16, 64, BF)
    for sources, n in (([0, 3, 0], 1), ([7, 1 << 30, 2], 2)):
        *_, want = run_fork(table, [20, 40, 10], sources, free, 16, host, dev)
        assert want[4] == n
    *_, want = run_fork(table, [20, 40, 10], [-1, -(1 << 31), 2], free, 16, host, dev)
    assert want[4] == 0


def test_pages_and_lengths_outside():
    """Ids outside the pool count for nothing and are no addresses; a length past its
    row of the table is held to it."""
    rng = np.random.default_rng(9)
    table, free, P = batch(rng, 3, 16, [40, 33, 20], 5)
    table[1][0], table[2][1] = P, -1
    host, dev = pools_of(rng, 1, P, 1, 16, 64, BF)
    t, n, f, c = i32(table), i32([40, 33, 1000]), i32(free + [0] * (P - len(free))), i32([len(free)])
    handle = ops.page_pools(dev)
    assert int(ops.paged_fork(t, n, i32([1, 1, 1]), f, c, handle)) == 0
    assert n.tolist() == [33] * 3 and t[:, 0].tolist() == [P] * 3
    t, n = i32([[3, 99, 0], [1, 2, -7], [-1, 5, 6]]), i32([48, 33, 1000])
    assert int(ops.paged_compact(t, n, f, c, handle)) == len({3, 0, 1, 2, 5, 6})
    assert t.tolist() == [[3, 99, 0], [1, 2, -7], [-1, 5, 4]]


@pytest.mark.parametrize("R,page,hi,share,HK,D,layers,dt,spare", [
    (1, 16, 0, 0, 1, 64, 1, BF, 5), (1, 16, 40, 0, 1, 64, 1, BF, 0), (5, 32, 300, 2, 2, 64, 2, FP, 33),
    (48, 64, 500, 3, 8, 128, 2, BF, 150), (700, 16, 200, 0, 1, 64, 1, BF, 5000),
    (3, 256, 2000, 1, 4, 128, 1, FP, 1),
])
def test_compact(R, page, hi, share, HK, D, layers, dt, spare):
    rng = np.random.default_rng(R * 17 + page)
    kv = rng.integers(0, hi + 1, R).tolist()
    table, free, P = batch(rng, R, page, kv, spare, share)
    host, dev = pools_of(rng, 2 * layers, P, HK, page, D, dt)
    padded = free + [-5] * (P + 2 - len(free))
    want = compact_by_hand(table, kv, padded, len(free), page, host)
    t, n, f, c = i32(table), i32(kv), i32(padded), i32([len(free)])
    handle = ops.page_pools(dev)
    for _ in range(2):  # the second time nothing moves
        live = ops.paged_compact(t, n, f, c, handle)
        assert t.tolist() == want[0] and n.tolist() == kv
        assert f.tolist() == want[1] and int(c) == want[2] and int(live) == want[3]
        same_pools(dev, want[4])


def test_a_pool_past_32_bits():
    """Pages whose offsets need more than 32 bits."""
    P, page = 3000, 256
    pool = torch.zeros((P, 32, page, 128), dtype=torch.float32, device=DEV)  # 12.6 GB
    pool[2990, 31, :9] = 7.0
    pool[2991, 5] = 3.0
    t, n = i32([[2991, 2990], [0, 0]]), i32([256 + 9, 0])
    f, c = i32(list(range(2000, 2999)) + [0] * 2001), i32([999])
    handle = ops.page_pools([pool])
    assert int(ops.paged_fork(t, n, i32([0, 0]), f, c, handle)) == 0
    assert t.tolist() == [[2991, 2990], [2991, 2998]] and n.tolist() == [265, 265]
    assert torch.equal(pool[2998, 31, :9], pool[2990, 31, :9]) and not pool[2998, 31, 9:].any()
    assert int(ops.paged_compact(t, n, f, c, handle)) == 3
    assert t.tolist() == [[1, 0], [1, 2]]
    assert (pool[1, 5] == 3.0).all() and (pool[2, 31, :9] == 7.0).all()


def test_many_pages():
    """A pool of as many pages as there may be, of few bytes each."""
    P = 1 << 20
    pool = torch.zeros((P, 1, 16, 8), dtype=torch.bfloat16, device=DEV)
    ids = [P - 1, 5, P - 32, P // 2, 31, 32]
    for i, p in enumerate(ids):
        pool[p] = i + 1
    t, n = i32([ids[:3], ids[3:]]), i32([48, 40])
    f, c = torch.zeros(P, dtype=torch.int32, device=DEV), i32([0])
    handle = ops.page_pools([pool])
    assert int(ops.paged_fork(t, n, i32([0, -1]), f, c, handle)) == 0
    assert f[:3].tolist() == [31, 32, P // 2] and int(c) == 3 and n.tolist() == [48, 0]
    n.copy_(i32([48, 40]))
    assert int(ops.paged_compact(t, n, f, c, handle)) == 6 and int(c) == P - 6
    assert sorted(sum(t.tolist(), [])) == list(range(6))
    assert [int(pool[p, 0, 0, 0]) for row in t.tolist() for p in row] == [1, 2, 3, 4, 5, 6]
    assert f[P - 7] == 6 and f[0] == P - 1


def test_graph_and_eager_alternate():
    """A fork and a compaction captured together, replayed from other lengths, with eager
    ones between."""
    rng = np.random.default_rng(11)
    page, R, W = 16, 6, 8
    pools = [torch.zeros((60, 2, page, 64), dtype=BF, device=DEV) for _ in range(4)]
    handle = ops.page_pools(pools)

    def start(seed):
        g = np.random.default_rng(seed)
        kv = g.integers(0, W * page + 1, R).tolist()
        table, free, _ = batch(g, R, page, kv, 60 - sum(-(-n // page) for n in kv), W=W)
        src = g.integers(-1, R, R).tolist()
        data = [torch.from_numpy(g.standard_normal(p.shape)).to(DEV).to(BF) for p in pools]
        return (i32(table), i32(kv), i32(src), i32(free + [0] * (60 - len(free))), i32([len(free)]),
                data)

    def both(t, n, s, f, c):
        return (ops.paged_fork(t, n, s, f, c, handle), ops.paged_compact(t, n, f, c, handle))

    def fill(data):
        for p, d in zip(pools, data):
            p.copy_(d)

    *static, data = start(0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with hip.graph_workspaces(), torch.cuda.graph(graph):
        out = both(*static)
    for seed in range(1, 6):
        *a, data = start(seed)
        for x, y in zip(static, a):
            x.copy_(y)
        fill(data)
        graph.replay()
        got = [v.clone() for v in (*static, *out, *pools)]
        fill(data)
        res = both(*a)
        assert all(torch.equal(x, y) for x, y in zip(got, (*a, *res, *pools))), seed
