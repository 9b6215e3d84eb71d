"""Operators of several continuations of one prompt over a paged key/value cache
(beam search, parallel samples, requests behind one system prompt), with what each
has to compute written out in elementary torch operations.

A case's ``op`` names the operator:

  select     beam search's choice: the likeliest continuations over the beams and the
             vocabulary of each prompt (``ops.beam_select``)
  fork       requests that go on from others' keys: full pages shared, part-filled
             ones copied in every layer, what nobody holds given back
             (``ops.paged_fork`` over ``ops.page_pools``)
  compact    the pages in use moved to the lowest ids of the pools
             (``ops.paged_compact``)
  shared     the leading keys that a group's requests hold in the same pages, and the
             step's work for all layers (``ops.paged_shared_plan``)
  attention  attention of requests behind shared prefixes, whose keys are read once for
             a group (``ops.paged_shared_attention``)

``own`` chooses between the plain forms and the library's calls. The sizes of a case's
groups and requests follow from its ``mix`` number, everything else from the seed.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
PKG = str(Path(__file__).resolve().parent.parent / "metal-autotune_amd")


def _ops():
    """The library's ops (the only import of the package)."""
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    from autotuner_runtime import ops
    return ops


# ---------------------------------------------------------------------------
# cases


def listed():
    return [
        # One prompt searched with four beams: latency.
        {"name": "select 1 x 4", "op": "select", "R": 1, "B": 4, "K": 4, "V": 151936,
         "masked": 0.0, "ended": 0.0, "dtype": "bfloat16"},
        # 37 prompts of five beams under a grammar that forbids most tokens; twice as
        # many continuations are kept as there are beams, a quarter of which have ended;
        # an odd vocabulary, fp16.
        {"name": "select 37 x 5 masked", "op": "select", "R": 37, "B": 5, "K": 10, "V": 65537,
         "masked": 0.9, "ended": 0.25, "dtype": "float16"},
        # Many prompts of eight beams, late in their search: HBM.
        {"name": "select 32 x 8", "op": "select", "R": 32, "B": 8, "K": 8, "V": 151936,
         "masked": 0.0, "ended": 0.1, "dtype": "bfloat16"},
        # Four beams of one prompt after a selection, few layers: latency.
        {"name": "fork 1 x 4", "op": "fork", "R": 1, "B": 4, "kv_lo": 900, "kv_hi": 1001,
         "page": 16, "layers": 2, "HK": 8, "D": 64, "dies": 0.5, "mix": 1, "dtype": "bfloat16"},
        # Eight prompts of eight beams, half of them replaced, twelve layers.
        {"name": "fork 8 x 8", "op": "fork", "R": 8, "B": 8, "kv_lo": 300, "kv_hi": 1500,
         "page": 64, "layers": 12, "HK": 8, "D": 128, "dies": 0.5, "mix": 2, "dtype": "bfloat16"},
        # A small batch's pool with holes.
        {"name": "compact 5", "op": "compact", "R": 5, "kv_lo": 1, "kv_hi": 300, "page": 32,
         "layers": 2, "HK": 2, "D": 64, "spare": 0.8, "mix": 3, "dtype": "float16"},
        # A long-running batch's, twelve layers.
        {"name": "compact 48", "op": "compact", "R": 48, "kv_lo": 1, "kv_hi": 1200, "page": 64,
         "layers": 12, "HK": 8, "D": 128, "spare": 0.6, "mix": 4, "dtype": "bfloat16"},
        # What four beams share.
        {"name": "shared 1 x 4", "op": "shared", "groups": 1, "per": 4, "pre_lo": 1001,
         "pre_hi": 1001, "tail": 40, "q": 1, "page": 64, "H": 32, "HK": 8, "D": 128, "mix": 5},
        # What 40 groups of up to 12 requests share, small pages.
        {"name": "shared 40 x 12", "op": "shared", "groups": 40, "per": 12, "pre_lo": 100,
         "pre_hi": 9000, "tail": 700, "q": 3, "page": 16, "H": 32, "HK": 8, "D": 128, "mix": 6},
        # Four beams of one prompt a thousand tokens in: latency.
        {"name": "attention 1 x 4", "op": "attention", "groups": 1, "per": 4, "pre_lo": 1001,
         "pre_hi": 1001, "tail": 40, "q": 1, "page": 64, "H": 32, "HK": 8, "D": 128, "mix": 7,
         "dtype": "bfloat16"},
        # Conversations behind five system prompts of different lengths, answers under
        # way; heads of 64, fp16, small pages.
        {"name": "attention 5 x 16", "op": "attention", "groups": 5, "per": 16, "pre_lo": 700,
         "pre_hi": 6000, "tail": 900, "q": 1, "page": 16, "H": 32, "HK": 8, "D": 64, "mix": 8,
         "dtype": "float16"},
        # 96 samples of answers to questions about one long document, up to four tokens
        # a step.
        {"name": "attention 1 x 96 long", "op": "attention", "groups": 1, "per": 96,
         "pre_lo": 16300, "pre_hi": 16300, "tail": 1500, "q": 4, "page": 64, "H": 32, "HK": 8,
         "D": 128, "mix": 9, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm; odd ones among them."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["select", "select", "fork", "compact", "shared", "attention", "attention"])
    dt = rng.choice(["bfloat16", "float16"])
    page = rng.choice([16, 32, 64, 128, 256])
    mix = rng.randrange(1 << 30)
    if op == "select":
        V, B = rng.choice([32000, 65536, 65537, 128257, 151936]), _log(rng, 1, 16)
        dt = rng.choice([dt, dt, "float32"])
        return {"op": op, "R": _log(rng, 1, max(1, 200 // B)), "B": B,
                "K": rng.choice([B, B, 2 * B, _log(rng, 1, 40)]), "V": V,
                "masked": rng.choice([0.0, 0.0, 0.5, 0.99]), "ended": rng.choice([0.0, 0.3]),
                "dtype": dt}
    heads = {"HK": rng.choice([1, 2, 4, 8]), "D": rng.choice([64, 128])}
    if op in ("fork", "compact"):
        B = _log(rng, 1, 16) if op == "fork" else 1
        R = _log(rng, 1, 64 // B)
        c = {"op": op, "R": R, "kv_lo": rng.choice([0, 1, 100]),
             "kv_hi": _log(rng, 101, max(102, 50000 // (R * B))), "page": page,
             "layers": rng.randint(1, 8), **heads, "mix": mix, "dtype": dt}
        if op == "fork":
            return {**c, "B": B, "dies": rng.choice([0.2, 0.5, 0.9])}
        return {**c, "spare": rng.choice([0.1, 0.5, 2.0])}
    groups = _log(rng, 1, 24)
    per = _log(rng, 1, max(2, 96 // groups))
    c = {"op": op, "groups": groups, "per": per, "tail": _log(rng, 1, 1000),
         "q": rng.choice([1, 1, 1, 4, 40]), "page": page, **heads, "mix": mix}
    c["H"] = c["HK"] * rng.choice([1, 2, 4, 5, 8]) if c["HK"] < 8 else 32
    c["pre_hi"] = _log(rng, 60, min(16000, 600000 // (groups * per)))
    c["pre_lo"] = rng.choice([1, c["pre_hi"] // 2, c["pre_hi"]])
    if op == "shared":
        return {**c, "per": max(2, per), "pre_hi": max(c["pre_hi"], 20 * page)}
    return {**c, "dtype": dt}


def _pages(n, page):
    return -(-n // page)


def _groups(case):
    """Of each group its requests' (prefix keys, keys after the step, new tokens): the
    first group is the largest and longest."""
    r = random.Random(case["mix"])
    out = []
    for g in range(case["groups"]):
        size = case["per"] if g == 0 else r.randint(max(1, case["per"] // 2), case["per"])
        pre = case["pre_hi"] if g == 0 else r.randint(case["pre_lo"], case["pre_hi"])
        q = [r.randint(1, case["q"]) for _ in range(size)]
        q[0] = case["q"] if g == 0 else q[0]
        out.append([(pre, pre + r.randint(0, case["tail"]) + n, n) for n in q])
    return out


def _kv(case):
    """Keys of each request of a fork (each prompt's beams are as long) or compaction."""
    r = random.Random(case["mix"])
    kv = [case["kv_hi"]] + [r.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["R"] - 1)]
    return [n for n in kv for _ in range(case.get("B", 1))]


def _sources(case):
    """The beam that each goes on from: some beams go on, the others are replaced by
    one of those of their prompt."""
    r = random.Random(case["mix"] + 1)
    out = []
    for p in range(case["R"]):
        B = case["B"]
        alive = [b for b in range(B) if r.random() >= case["dies"]] or [r.randrange(B)]
        out += [p * B + (b if b in alive else r.choice(alive)) for b in range(B)]
    return out


# ---------------------------------------------------------------------------
# inputs


def _state(table, kv, free, capacity):
    """Table, lengths, free list and its count in one array, so that a pass can begin
    with what it was given: (array, views)."""
    R, W = table.shape
    parts = [table.reshape(-1), kv, torch.nn.functional.pad(free, (0, capacity - free.numel())),
             torch.tensor([free.numel()], dtype=torch.int32, device=DEV)]
    buf = torch.cat([p.to(torch.int32) for p in parts])
    t, lens, fp, n = torch.split(buf, [R * W, R, capacity, 1])
    return buf, {"table": t.view(R, W), "kv": lens, "free": fp, "free_count": n}


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op = case["op"]

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    def rand(dt, *shape):
        return torch.empty(shape, dtype=dt, device=DEV).normal_(generator=gen)

    if op == "select":
        R, B, V, dt = case["R"], case["B"], case["V"], DTYPES[case["dtype"]]
        # a few likely tokens over a broad tail, others a beam; under a grammar the
        # forbidden ones are -inf (the first stays allowed)
        x = 2.5 * torch.randn((R * B, V), generator=gen, device=DEV)
        hot = torch.randint(0, V // 8, (R * B, 8), generator=gen, device=DEV)
        hot += V // 8 * torch.arange(8, device=DEV)
        x.scatter_add_(1, hot, 4 + 6 * torch.rand((R * B, 8), generator=gen, device=DEV))
        if case["masked"]:
            gone = torch.rand((R * B, V), generator=gen, device=DEV) < case["masked"]
            gone[:, 0] = False
            gone.scatter_(1, hot[:, :1], False)
            x.masked_fill_(gone, float("-inf"))
        scores = -20 - 3 * torch.rand((R, B), generator=gen, device=DEV)
        return {"case": case, "x": x.to(dt), "scores": scores,
                "ended": torch.rand((R, B), generator=gen, device=DEV) < case["ended"],
                "eos": V - 7}
    if op in ("fork", "compact"):
        kv, page, dt = _kv(case), case["page"], DTYPES[case["dtype"]]
        counts = [_pages(n, page) for n in kv]
        live, R = sum(counts), len(kv)
        W = max(1, max(counts))
        # room for a copy a request, or as many holes as the case says
        P = live + (R + 3 if op == "fork" else 1 + int(case["spare"] * live))
        order = torch.randperm(P, generator=gen, device=DEV)
        n = i32(counts)
        w = torch.arange(W, device=DEV)
        at = (torch.cumsum(n, 0) - n)[:, None] + w
        table = torch.where(w < n[:, None], order[at.clamp(max=P - 1)], 0)
        buf, views = _state(table, i32(kv), order[live:], P)
        pools = [rand(dt, P, case["HK"], page, case["D"]) for _ in range(2 * case["layers"])]
        st = {"case": case, "buf": buf, "given": buf.clone(), **views, "pools": pools,
              "page": page}
        if op == "fork":
            st["sources"] = i32(_sources(case))
        if own:
            st["handle"] = _ops().page_pools(pools)
        return st
    groups, page = _groups(case), case["page"]
    rows, cu_groups, pool = [], [0], 0
    kv, q, pre = [], [], []
    at = random.Random(seed)
    for requests in groups:
        shared = requests[0][0] // page  # (what the prefix's last page holds is copied)
        if op == "shared":  # the requests have parted somewhere behind its half
            shared = at.randint(shared // 2, shared)
        first, pool = pool, pool + shared
        for p, n, new in requests:
            own_pages = _pages(n, page) - shared
            rows.append(list(range(first, first + shared)) + list(range(pool, pool + own_pages)))
            pool += own_pages
            kv.append(n)
            q.append(new)
        pre.append(shared * page)
        cu_groups.append(len(rows))
    W, pool = max(len(r) for r in rows), max(1, pool)
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.zeros((len(rows), W), dtype=torch.int32)
    for r, ids in enumerate(rows):
        table[r, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    cu = [0]
    for n in q:
        cu.append(cu[-1] + n)
    st = {"case": case, "table": order[table.to(DEV).long()], "kv": i32(kv), "cu": i32(cu),
          "cu_groups": i32(cu_groups), "T": cu[-1], "most_q": max(q), "page": page}
    if op == "shared":
        return st
    dt, H, HK, D = DTYPES[case["dtype"]], case["H"], case["HK"], case["D"]
    st.update({"q": rand(dt, cu[-1], H, D), "k": rand(dt, pool, HK, page, D),
               "v": rand(dt, pool, HK, page, D), "scale": D ** -0.5})
    if own:  # made once a step, for the attention of every layer
        st["plan"] = _shared_plan(st)
    return st


def _shared_plan(st):
    case = st["case"]
    return _ops().paged_shared_plan(st["table"], st["cu"], st["kv"], st["cu_groups"], st["page"],
                                    st["T"], case["H"], case["HK"], case["D"])


# ---------------------------------------------------------------------------
# one pass


def _plain_select(st):
    # in 64 bits: candidates of different beams lie close together
    R, B = st["scores"].shape
    x, V, K = st["x"].double(), st["case"]["V"], st["case"]["K"]
    m = x.amax(-1, keepdim=True)
    c = x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
    del x
    c = c.view(R, B, V) + st["scores"].double()[..., None]
    ended, eos = st["ended"], st["eos"]
    c.masked_fill_(ended[..., None], float("-inf"))
    c[..., eos] = torch.where(ended, st["scores"].double(), c[..., eos])
    values, at = torch.sort(c.view(R, B * V), dim=-1, descending=True, stable=True)
    values, at = values[:, :K], at[:, :K]
    there = values > float("-inf")
    parents = torch.where(there, at // V, 0) + B * torch.arange(R, device=DEV)[:, None]
    tokens = torch.where(there, at % V, 0)
    done = there & (ended.view(-1)[parents] | (tokens == eos))
    return {"scores": values.float(), "parents": parents.int(), "tokens": tokens.int(),
            "finished": done}


def _marks(table, pages, P):
    """Which pages the first ``pages`` entries of the table's rows name."""
    live = torch.arange(table.shape[1], device=DEV) < pages[:, None]
    marks = torch.zeros(P + 1, dtype=torch.long, device=DEV)
    marks.scatter_(0, torch.where(live, table.long(), P).view(-1), 1)
    return marks[:P] > 0


def _plain_fork(st):
    page, table, kv, free, count = (st[k] for k in ("page", "table", "kv", "free", "free_count"))
    R, W = table.shape
    P = st["pools"][0].shape[0]
    s, r = st["sources"].long(), torch.arange(R, device=DEV)
    alive, src = s >= 0, s.clamp(min=0)
    pages = (kv.long() + page - 1) // page
    new_kv = torch.where(alive, kv.long()[src], 0)
    new_pages = (new_kv + page - 1) // page
    rows = table.long()[src]
    # pages that nobody holds any more, pushed in the order of their ids
    gone = _marks(table, pages, P) & ~_marks(rows, new_pages, P)
    at = torch.where(gone, count.long() + torch.cumsum(gone, 0) - 1, P)
    pushed = torch.cat([free.long(), free.new_zeros(1).long()])
    pushed.scatter_(0, at, torch.arange(P, device=DEV))
    n = count.long() + gone.sum()
    # a part-filled page stays with one child, itself or the first
    keeper = torch.full((R,), R, device=DEV).scatter_reduce(0, torch.where(alive, src, 0),
                                                            torch.where(alive, r, R), "amin")
    keeper = torch.where(s == r, r, keeper)
    copy = alive & (new_kv % page != 0) & (keeper[src] != r)
    taken = torch.cumsum(copy, 0)
    lacking = (taken[-1] - n).clamp(min=0)
    ok = lacking == 0
    copy = copy & ok
    last = (new_pages - 1).clamp(min=0)
    old = rows.gather(1, last[:, None])[:, 0]
    new = torch.where(copy, pushed[(n - taken).clamp(0, P - 1)], old)
    rows = rows.scatter(1, last[:, None], new[:, None])
    inside = torch.arange(page, device=DEV) < torch.where(copy, new_kv % page, 0)[:, None]
    inside = inside[:, None, :, None]
    for pool in st["pools"]:
        pool[new] = torch.where(inside, pool[old], pool[new])
    write = ok & (torch.arange(W, device=DEV) < new_pages[:, None])
    table.copy_(torch.where(write, rows, table.long()))
    kv.copy_(torch.where(ok, new_kv, kv.long()))
    free.copy_(torch.where(ok, pushed[:P], free.long()))
    count.copy_(torch.where(ok, n - copy.sum(), count.long()))
    return lacking.int().view(1)


def _plain_compact(st):
    page, table, kv, free, count = (st[k] for k in ("page", "table", "kv", "free", "free_count"))
    P, W = st["pools"][0].shape[0], table.shape[1]
    pages = (kv.long() + page - 1) // page
    live = _marks(table, pages, P)
    n, ids = live.sum(), torch.arange(P, device=DEV)
    hole, move = ~live & (ids < n), live & (ids >= n)
    spare = torch.full((P + 1,), P, device=DEV)
    holes = spare.scatter(0, torch.where(hole, torch.cumsum(hole, 0) - 1, P), ids)
    to = torch.where(move, holes[(torch.cumsum(move, 0) - 1).clamp(min=0)], ids)
    back = torch.cat([ids, ids[:1]]).scatter(0, torch.where(move, to, P), ids)[:P]
    for pool in st["pools"]:
        pool.copy_(pool[back])
    live_entry = torch.arange(W, device=DEV) < pages[:, None]
    table.copy_(torch.where(live_entry, to[table.long()], table.long()))
    free.copy_(torch.where(ids < P - n, P - 1 - ids, free.long()))
    count.copy_(P - n)
    return n.int().view(1)


def _plain_shared(st):
    table, kv, cu, page = st["table"], st["kv"].long(), st["cu"].long(), st["page"]
    R, W = table.shape
    G = st["cu_groups"].numel() - 1
    r = torch.arange(R, device=DEV)
    group = torch.searchsorted(st["cu_groups"][1:].long(), r, right=True)
    n = cu[1:] - cu[:-1]
    takes_part = (n > 0) & (kv > 0)
    lead = torch.full((G,), R, device=DEV).scatter_reduce(
        0, group, torch.where(takes_part, r, R), "amin")
    same = table == table[lead.clamp(max=R - 1)[group]]
    alike = torch.cumprod(same.long(), 1).sum(1)
    alike = torch.minimum(alike, (kv - n).clamp(min=0) // page)
    most = torch.full((G,), W, device=DEV).scatter_reduce(
        0, group, torch.where(takes_part, alike, W), "amin")
    return {"keys": (torch.where(lead < R, most, 0) * page).int()}


def _plain_attention(st):
    case, q, table, cu, kv = st["case"], st["q"], st["table"].long(), st["cu"].long(), st["kv"].long()
    T, H, D = q.shape
    R, HK, page = table.shape[0], case["HK"], case["page"]
    G, Lq = H // HK, st["most_q"]
    L = table.shape[1] * page
    n = cu[1:] - cu[:-1]
    i = torch.arange(Lq, device=DEV)
    rows = (cu[:-1, None] + i).clamp(max=T - 1)
    # [R, HK, G Lq, D] against [R, HK, L, D]
    qq = q[rows].float().reshape(R, Lq, HK, G, D).permute(0, 2, 3, 1, 4).reshape(R, HK, G * Lq, D)
    k = st["k"][table].permute(0, 2, 1, 3, 4).reshape(R, HK, L, D).float()
    s = torch.matmul(qq, k.transpose(-1, -2)).reshape(R, HK, G, Lq, L) * st["scale"]
    del k, qq
    j = torch.arange(L, device=DEV)
    seen = j <= (kv - n)[:, None, None] + i[:, None]
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(s - m)
    del s
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0).reshape(R, HK, G * Lq, L)
    v = st["v"][table].permute(0, 2, 1, 3, 4).reshape(R, HK, L, D).float()
    o = torch.matmul(p, v).reshape(R, HK, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(R, Lq, H, D)
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True)
    return o[r, t - cu[r]].to(q.dtype)


def run(st):
    case = st["case"]
    op = case["op"]
    if op in ("fork", "compact"):
        # both change what they are given: every pass begins with the same
        st["buf"].copy_(st["given"])
        if not own:
            n = (_plain_fork if op == "fork" else _plain_compact)(st)
        elif op == "fork":
            n = _ops().paged_fork(st["table"], st["kv"], st["sources"], st["free"],
                                  st["free_count"], st["handle"])
        else:
            n = _ops().paged_compact(st["table"], st["kv"], st["free"], st["free_count"],
                                     st["handle"])
        return {"refused" if op == "fork" else "live": n, "table": st["table"], "kv": st["kv"],
                "free": st["free"], "free_count": st["free_count"], "pools": st["pools"]}
    if not own:
        return {"select": _plain_select, "shared": _plain_shared,
                "attention": _plain_attention}[op](st)
    ops = _ops()
    if op == "select":
        s = ops.beam_select(st["x"], st["scores"], case["K"], st["ended"], st["eos"])
        return {"scores": s.scores, "parents": s.parents, "tokens": s.tokens,
                "finished": s.finished}
    if op == "shared":
        return {"keys": _shared_plan(st).keys}
    return ops.paged_shared_attention(st["q"], st["k"], st["v"], st["table"], st["plan"],
                                      st["scale"])


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "select":
        size = 4 if case["dtype"] == "float32" else 2
        R, B, K, V = case["R"], case["B"], case["K"], case["V"]
        # (the logits of beams that have ended are not needed; which, the seed says)
        rows = R * B * (1 - case["ended"])
        return {"bytes": int(rows * V * size) + 5 * R * B + 13 * R * K, "flops": int(3 * rows * V)}
    if op in ("fork", "compact"):
        kv, page = _kv(case), case["page"]
        R, counts = len(kv), [_pages(n, page) for n in kv]
        row = 2 * case["layers"] * case["HK"] * case["D"] * 2  # bytes of a key in all pools
        if op == "fork":
            src = _sources(case)
            # every child but one of a beam copies its part-filled page; tables are read
            # and the replaced rows written, freed pages pushed
            rows = sum(kv[s] % page for r, s in enumerate(src) if s != r)
            changed = sum(counts[s] for r, s in enumerate(src) if s != r)
            return {"bytes": 2 * row * rows + 4 * (sum(counts) + 2 * changed + 4 * R), "flops": 0}
        live = sum(counts)
        # the share of the pages in use whose id is past their number
        moved = int(live * (1 - live / (live + 1 + int(case["spare"] * live))))
        free = 1 + int(case["spare"] * live)
        return {"bytes": 2 * row * page * moved + 4 * (2 * live + R + free), "flops": 0}
    groups, page = _groups(case), case["page"]
    shared = [g[0][0] // page for g in groups]
    R = sum(len(g) for g in groups)
    if op == "shared":
        # (the seed says where in the prefix's second half the requests part)
        return {"bytes": 3 * sum(n * len(g) for n, g in zip(shared, groups)) +
                4 * (3 * R + 2 * len(groups)), "flops": 0}
    H, HK, D = case["H"], case["HK"], case["D"]
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for g in groups for _, k, n in g)
    keys = sum(page * s + sum(k - page * s for _, k, _ in g) for s, g in zip(shared, groups))
    tokens = sum(n for g in groups for _, _, n in g)
    return {"bytes": 2 * D * (2 * H * tokens + 2 * HK * keys) + 4 * (keys // page + 2 * R),
            "flops": 4 * H * D * pairs}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    op, f64 = case["op"], torch.float64
    if op in ("fork", "compact", "shared"):
        return None  # whole numbers and moved values: the plain form's are the definition's
    st = prepare(case, seed)
    if op == "select":
        R, B, K, V = case["R"], case["B"], case["K"], case["V"]
        out = torch.empty((R, K), dtype=f64, device=DEV)
        for r in range(R):
            rows = torch.log_softmax(st["x"][r * B:(r + 1) * B].to(f64), -1)
            rows += st["scores"][r].to(f64)[:, None]
            ended = st["ended"][r]
            best = torch.cat([rows[~ended].reshape(-1), st["scores"][r][ended].to(f64),
                              torch.full((K,), -math.inf, dtype=f64, device=DEV)])
            out[r] = torch.topk(best, K).values
        return {"scores": out, "parents": None, "tokens": None, "finished": None}
    H, HK, D = case["H"], case["HK"], case["D"]
    G = H // HK
    out = torch.zeros(st["q"].shape, dtype=f64, device=DEV)
    cu, kv = st["cu"].tolist(), st["kv"].tolist()
    for r, n in enumerate(kv):
        a, b = cu[r], cu[r + 1]
        pages = st["table"][r, :_pages(n, case["page"])].long()
        last = n - (b - a)  # the first new token's position
        k = st["k"][pages].transpose(0, 1).reshape(HK, -1, D)[:, :n].to(f64)
        v = st["v"][pages].transpose(0, 1).reshape(HK, -1, D)[:, :n].to(f64)
        hide = torch.ones((b - a, n), dtype=torch.bool, device=DEV).triu(last + 1)
        for h in range(HK):
            for g in range(h * G, h * G + G):
                s = st["q"][a:b, g].to(f64) @ k[h].T * st["scale"]
                s[hide] = -math.inf
                out[a:b, g] = torch.softmax(s, -1) @ v[h]
    return out
