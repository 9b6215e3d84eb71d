"""Operators of serving several requests at once over a paged key/value cache,
with what each has to compute written out in elementary torch operations.

A case's ``op`` names the operator:

  plan       one step's bookkeeping on the GPU, from the requests' lengths:
             new pages taken from the free list into the block table, and for
             every token of the step its position and its cache slot
             (``ops.paged_plan``)
  prologue   q/k RMSNorm + RoPE at each token's own position, q returned, k and
             v written into the pages at each token's slot
             (``ops.norm_rope_paged``, ``ops.rope_table``)
  attention  causal GQA attention of every request's new tokens over its pages:
             one token a request (decode), chunks of prompts, or both in one
             call (``ops.paged_attention``)
  logprobs   log probabilities of given tokens, the entropy of each row and its
             most probable tokens (``ops.token_logprobs``)

``own`` chooses between the plain forms and the library's calls. The lengths of
a case's requests follow from its ``mix`` number, their order and everything
else from the seed.
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
EPS = 1e-6
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
        # A decode step's bookkeeping for 32 running conversations.
        {"name": "plan decode 32", "op": "plan", "R": 32, "kv_lo": 100, "kv_hi": 8191, "page": 64,
         "chunks": 0, "q_hi": 1, "spare": 0, "mix": 1},
        # A large mixed step: 256 requests of which a quarter bring prompt
        # chunks, in a token buffer with room left.
        {"name": "plan mixed 256", "op": "plan", "R": 256, "kv_lo": 1, "kv_hi": 16384, "page": 16,
         "chunks": 64, "q_hi": 501, "spare": 77, "mix": 2},
        # 37 decoding requests far into their contexts; half the head is
        # rotated, in interleaved pairs, fp16, 32/8 heads of 64.
        {"name": "prologue decode 37 far", "op": "prologue", "T": 37, "H": 32, "HK": 8, "D": 64,
         "dims": 32, "interleaved": True, "base": 1e6, "scale": 0.25, "pos_lo": 90000,
         "pos_hi": 131072, "page": 32, "dtype": "float16"},
        # The chunks of several prompts, 8192 tokens in all, 32/8 heads of 128.
        {"name": "prologue prefill 8192", "op": "prologue", "T": 8192, "H": 32, "HK": 8, "D": 128,
         "dims": 128, "interleaved": False, "base": 1e6, "scale": 1.0, "pos_lo": 0,
         "pos_hi": 8192, "page": 64, "dtype": "bfloat16"},
        # One conversation decoding, a thousand tokens in: latency.
        {"name": "attention decode 1 x 1001", "op": "attention", "R": 1, "H": 32, "HK": 8,
         "D": 128, "kv_lo": 1001, "kv_hi": 1001, "chunks": 0, "q_hi": 1, "page": 64, "mix": 3,
         "dtype": "bfloat16"},
        # 48 conversations of very different lengths decoding together.
        {"name": "attention decode 48 ragged", "op": "attention", "R": 48, "H": 32, "HK": 8,
         "D": 128, "kv_lo": 64, "kv_hi": 8191, "chunks": 0, "q_hi": 1, "page": 32, "mix": 4,
         "dtype": "bfloat16"},
        # Three long documents being answered, 32/8 heads of 64, fp16.
        {"name": "attention decode 3 long", "op": "attention", "R": 3, "H": 32, "HK": 8, "D": 64,
         "kv_lo": 40000, "kv_hi": 65521, "chunks": 0, "q_hi": 1, "page": 128, "mix": 5,
         "dtype": "float16"},
        # A step that decodes 16 requests beside 4 prompt chunks behind cached
        # prefixes, small pages.
        {"name": "attention mixed step", "op": "attention", "R": 20, "H": 32, "HK": 8, "D": 128,
         "kv_lo": 300, "kv_hi": 4096, "chunks": 4, "q_hi": 512, "page": 16, "mix": 6,
         "dtype": "bfloat16"},
        # Four prompts of about 2048 tokens prefilled together.
        {"name": "attention prefill 4 x 2048", "op": "attention", "R": 4, "H": 32, "HK": 8,
         "D": 128, "kv_lo": 1500, "kv_hi": 2048, "chunks": 4, "q_hi": 2048, "page": 64, "mix": 7,
         "dtype": "bfloat16"},
        # The logits of one decode step, its token's log probability and the
        # five likeliest beside it.
        {"name": "logprobs 1 row top 5", "op": "logprobs", "rows": 1, "V": 151936, "top": 5,
         "masked": 0.0, "dtype": "bfloat16"},
        # 37 requests under a grammar that forbids most tokens, an odd
        # vocabulary, fp16.
        {"name": "logprobs 37 masked top 20", "op": "logprobs", "rows": 37, "V": 65537, "top": 20,
         "masked": 0.9, "dtype": "float16"},
        # A prompt scored: every position's token.
        {"name": "logprobs 1024 scored", "op": "logprobs", "rows": 1024, "V": 151936, "top": 1,
         "masked": 0.0, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm; odd ones among them."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "prologue", "attention", "attention", "logprobs"])
    dt = rng.choice(["bfloat16", "float16"])
    if op == "plan":
        R = _log(rng, 1, 400)
        return {"op": op, "R": R, "kv_lo": rng.choice([0, 1, 100]), "kv_hi": _log(rng, 200, 16384),
                "page": rng.choice([16, 32, 64, 128, 256]),
                "chunks": rng.choice([0, rng.randint(0, min(R, 24))]), "q_hi": _log(rng, 2, 600),
                "spare": rng.choice([0, rng.randint(1, 200)]), "mix": rng.randrange(1 << 30)}
    if op == "prologue":
        D, HK = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        lo = rng.choice([0, 0, 5000, 100000])
        T = _log(rng, 1, 6000)
        return {"op": op, "T": T, "H": HK * rng.choice([1, 2, 4, 5, 8]) if HK < 8 else 32, "HK": HK,
                "D": D, "dims": rng.choice([D, D, D // 2]), "interleaved": rng.random() < 0.4,
                "base": rng.choice([1e4, 1e6]), "scale": rng.choice([1.0, 0.25]), "pos_lo": lo,
                "pos_hi": lo + _log(rng, T + 1, 3 * T + 30000), "page": rng.choice([16, 32, 64, 128]),
                "dtype": dt}
    if op == "attention":
        D, HK = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        H = HK * rng.choice([1, 2, 4, 5, 8]) if HK < 8 else 32
        form = rng.choice(["decode", "decode", "few", "mixed", "prompts"])
        c = {"op": op, "H": H, "HK": HK, "D": D, "page": rng.choice([16, 32, 64, 128, 256]),
             "mix": rng.randrange(1 << 30), "dtype": dt}
        if form in ("decode", "few"):
            R = _log(rng, 1, 64)
            hi = _log(rng, 130, min(50000, 200000 // R))
            chunks = 0 if form == "decode" else R
            return {**c, "R": R, "kv_lo": rng.choice([1, hi // 2]), "kv_hi": hi, "chunks": chunks,
                    "q_hi": 1 if form == "decode" else rng.randint(2, 6)}
        if form == "mixed":
            R = rng.randint(3, 24)
            return {**c, "R": R, "kv_lo": 20, "kv_hi": _log(rng, 500, 4096),
                    "chunks": rng.randint(1, 4), "q_hi": _log(rng, 16, 450)}
        hi = _log(rng, 60, 1800)
        return {**c, "R": rng.randint(1, 4), "kv_lo": max(1, hi // 2), "kv_hi": hi, "chunks": 4,
                "q_hi": hi}
    V, dt = rng.choice([32000, 65536, 65537, 128257, 151936]), rng.choice([dt, dt, "float32"])
    return {"op": op, "rows": _log(rng, 1, 350 if dt == "float32" else 700), "V": V,
            "top": rng.choice([0, 1, 5, 20]), "masked": rng.choice([0.0, 0.0, 0.5, 0.99]),
            "dtype": dt}


def _lengths(case):
    """(keys of each request after the step, new tokens of each request). The
    first request is the longest; the requests that bring chunks come last."""
    r = random.Random(case["mix"])
    R, lo, hi = case["R"], case["kv_lo"], case["kv_hi"]
    kv = [hi] + [r.randint(lo, hi) for _ in range(R - 1)]
    q = [1] * R
    for i in range(max(0, R - case["chunks"]), R):
        kv[i] = max(kv[i], 1)
        q[i] = min(kv[i], case["q_hi"] if i == R - 1 else r.randint(max(1, case["q_hi"] // 2), case["q_hi"]))
    if case["op"] == "plan":
        return [k + n for k, n in zip(kv, q)], q  # kv: the keys before the step
    return [max(k, n) for k, n in zip(kv, q)], q


# ---------------------------------------------------------------------------
# inputs


def _pages(n, page):
    return -(-n // page)


def _block_table(kv, page, gen, spare=0):
    """Every request's pages, scattered over a pool that holds just them (and
    ``spare`` free ones): (table [R, most pages], the pool's pages, the free ones)."""
    counts = [_pages(n, page) for n in kv]
    total = sum(counts) + spare
    order = torch.randperm(max(1, total), generator=gen, device=DEV).to(torch.int32)
    width = max(1, max(counts))
    n = torch.tensor(counts, device=DEV)
    first = torch.cumsum(n, 0) - n
    w = torch.arange(width, device=DEV)
    at = (first[:, None] + w).clamp(max=max(1, total) - 1)
    table = torch.where(w < n[:, None], order[at], 0).to(torch.int32)
    return table, max(1, total), order[sum(counts):]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op = case["op"]

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    if op in ("plan", "attention"):
        kv, q = _lengths(case)
        order = list(range(len(kv)))
        random.Random(seed).shuffle(order)
        kv, q = [kv[i] for i in order], [q[i] for i in order]
        page = case["page"]
    if op == "plan":
        before = [k - n for k, n in zip(kv, q)]
        need = sum(_pages(k, page) - _pages(b, page) for k, b in zip(kv, before))
        table, _, free = _block_table(before, page, gen, need + 9)
        wide = torch.zeros((len(kv), max(_pages(k, page) for k in kv)), dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table[:, :wide.shape[1]]
        return {"case": case, "table": wide, "kv": i32(before), "q": i32(q), "free": free,
                "free_count": i32([free.numel()]), "page": page, "T": sum(q) + case["spare"]}
    if op == "attention":
        dt, H, HK, D = DTYPES[case["dtype"]], case["H"], case["HK"], case["D"]
        table, pool, _ = _block_table(kv, page, gen)
        cu = [0]
        for n in q:
            cu.append(cu[-1] + n)

        def rand(*shape):
            return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dt)

        return {"case": case, "q": rand(cu[-1], H, D), "k": rand(pool, HK, page, D),
                "v": rand(pool, HK, page, D), "table": table, "cu": i32(cu), "kv": i32(kv),
                "most_q": max(q), "most_kv": max(kv), "scale": D ** -0.5}
    if op == "prologue":
        dt, T, H, HK, D = DTYPES[case["dtype"]], case["T"], case["H"], case["HK"], case["D"]
        page = case["page"]
        pool = _pages(T, page) + 3
        # one projection's output, of which q, k and v are column ranges
        qkv = torch.randn((T, (H + 2 * HK) * D), generator=gen, device=DEV).to(dt)
        norms = [(1 + 0.1 * torch.randn(D, generator=gen, device=DEV)).to(dt) for _ in range(2)]
        cache = [torch.randn((pool, HK, page, D), generator=gen, device=DEV).to(dt) for _ in range(2)]
        span = case["pos_hi"] - case["pos_lo"]
        first = case["pos_lo"] + torch.randint(0, max(1, span - T + 1), (1,), generator=gen, device=DEV)
        i = torch.arange(case["dims"] // 2, device=DEV, dtype=torch.float64)
        return {"case": case, "q": qkv[:, :H * D], "k": qkv[:, H * D:(H + HK) * D],
                "v": qkv[:, (H + HK) * D:], "q_norm": norms[0], "k_norm": norms[1],
                "k_pages": cache[0], "v_pages": cache[1],
                "table": case["scale"] * case["base"] ** (-2 * i / case["dims"]),
                "positions": (first + torch.arange(T, device=DEV)).to(torch.int32),
                "slots": torch.randperm(pool * page, generator=gen, device=DEV)[:T].to(torch.int32)}
    dt, rows, V = DTYPES[case["dtype"]], case["rows"], case["V"]
    # a few likely tokens over a broad tail; under a grammar the forbidden ones
    # are -inf (the first stays allowed)
    x = 2.5 * torch.randn((rows, V), generator=gen, device=DEV)
    hot = torch.randint(0, V // 8, (rows, 8), generator=gen, device=DEV)
    hot += V // 8 * torch.arange(8, device=DEV)
    x.scatter_add_(1, hot, 4 + 6 * torch.rand((rows, 8), generator=gen, device=DEV))
    if case["masked"]:
        gone = torch.rand((rows, V), generator=gen, device=DEV) < case["masked"]
        gone[:, 0] = False
        gone.scatter_(1, hot[:, :1], False)
        x.masked_fill_(gone, float("-inf"))
        del gone
    return {"case": case, "x": x.to(dt), "tokens": hot[:, 0].contiguous()}


# ---------------------------------------------------------------------------
# one pass


def _plain_plan(st):
    page, T, table = st["page"], st["T"], st["table"]
    R, W = table.shape
    kv, q, free, count = st["kv"].long(), st["q"].long(), st["free"].long(), st["free_count"].long()
    old, new = (kv + page - 1) // page, (kv + q + page - 1) // page
    fits = new <= W
    need = torch.where(fits, new - old, 0)
    end = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (end <= count))
    cu = torch.cat([torch.zeros_like(q[:1]), torch.cumsum(q, 0)])
    # the pages taken, from the end of the free list, request after request
    w = torch.arange(W, device=DEV)
    at = count - 1 - ((end - need)[:, None] + w - old[:, None])
    taken = free[at.clamp(0, free.numel() - 1)]
    grown = torch.where(ok[:, None] & (w >= old[:, None]) & (w < new[:, None]), taken, table.long())
    t = torch.arange(T, device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True).clamp(max=R - 1)
    real = t < cu[-1]
    pos = kv[r] + t - cu[r]
    page_of = grown[r, (pos // page).clamp(0, W - 1)]
    slots = torch.where(real & ok[r], page_of * page + pos % page, -1)
    left = count - torch.where(ok, torch.where(need > 0, end, 0), 0).max()
    table.copy_(grown)
    i32 = torch.int32
    return {"cu_q": cu.to(i32), "kv_lens": torch.where(ok, kv + q, 0).to(i32),
            "positions": torch.where(real, pos, 0).to(i32), "slots": slots.to(i32),
            "free_count": left.to(i32), "refused": (~ok).sum().reshape(1).to(i32), "table": table}


def _plain_prologue(st):
    case = st["case"]
    T, D, dims = case["T"], case["D"], case["dims"]
    half = dims // 2
    angle = st["positions"].double()[:, None] * st["table"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x, norm):
        x = x.reshape(T, -1, D).float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.float()
        if case["interleaved"]:
            a, b = x[..., 0:dims:2], x[..., 1:dims:2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = x[..., :half], x[..., half:dims]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([y, x[..., dims:]], -1)

    dt = st["q"].dtype
    page, row = st["slots"].long() // case["page"], st["slots"].long() % case["page"]
    st["k_pages"][page, :, row] = turn(st["k"], st["k_norm"]).to(dt)
    st["v_pages"][page, :, row] = st["v"].reshape(T, -1, D)
    return {"q": turn(st["q"], st["q_norm"]).to(dt), "k_pages": st["k_pages"],
            "v_pages": st["v_pages"]}


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


def _plain_logprobs(st):
    x, k = st["x"].float(), st["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, e * (x - m), 0).sum(-1, keepdim=True) / total
    picked = x.gather(1, st["tokens"][:, None]) - lse
    out = {"logprobs": picked[:, 0], "entropy": entropy[:, 0]}
    if k:
        values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_ids"] = ids[:, :k].to(torch.int32)
        out["top_logprobs"] = values[:, :k] - lse
    return out


def run(st):
    case = st["case"]
    op = case["op"]
    if not own:
        return {"plan": _plain_plan, "prologue": _plain_prologue, "attention": _plain_attention,
                "logprobs": _plain_logprobs}[op](st)
    ops = _ops()
    if op == "plan":
        p = ops.paged_plan(st["table"], st["kv"], st["q"], st["free"], st["free_count"],
                           st["page"], st["T"])
        return {"cu_q": p.cu_q, "kv_lens": p.kv_lens, "positions": p.positions, "slots": p.slots,
                "free_count": p.free_count, "refused": p.refused, "table": st["table"]}
    if op == "prologue":
        q = ops.norm_rope_paged(st["q"], st["k"], st["v"], st["q_norm"], st["k_norm"], case["H"],
                                case["HK"], EPS, st["table"], st["positions"], st["slots"],
                                st["k_pages"], st["v_pages"], traditional=case["interleaved"])
        return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if op == "attention":
        return ops.paged_attention(st["q"], st["k"], st["v"], st["table"], st["cu"], st["kv"],
                                   st["scale"], max_q_len=st["most_q"])
    r = ops.token_logprobs(st["x"], st["tokens"], top=case["top"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if case["top"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    op = case["op"]
    if op == "plan":
        kv, q = _lengths(case)
        page, R, T = case["page"], case["R"], sum(q) + case["spare"]
        # entries of the block table that are read (the page a token continues)
        # and written, the free list's share, lengths, tokens
        started = sum((k - n) % page != 0 for k, n in zip(kv, q))
        need = sum(_pages(k, page) - _pages(k - n, page) for k, n in zip(kv, q))
        return {"bytes": 4 * (2 * R + started + 2 * need + 2 * R + 1 + 2 * T + 3), "flops": 0}
    if op == "prologue":
        T, H, HK, D, dims = case["T"], case["H"], case["HK"], case["D"], case["dims"]
        return {"bytes": 2 * (2 * T * (H + 2 * HK) * D + 2 * D) + 8 * T + 8 * (dims // 2),
                "flops": T * (H + HK) * (4 * D + 3 * dims)}
    if op == "attention":
        kv, q = _lengths(case)
        H, HK, D = case["H"], case["HK"], case["D"]
        pairs = sum(n * (k - n) + n * (n + 1) // 2 for k, n in zip(kv, q))
        pages = sum(_pages(k, case["page"]) for k in kv)
        return {"bytes": 2 * D * (2 * H * sum(q) + 2 * HK * sum(kv)) + 4 * (pages + 2 * len(kv) + 1),
                "flops": 4 * H * D * pairs}
    size = 4 if case["dtype"] == "float32" else 2
    rows, V, k = case["rows"], case["V"], case["top"]
    return {"bytes": rows * (V * size + 8 + 8 + 8 * k), "flops": 5 * rows * V}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "plan":
        return None  # whole numbers: the plain form's are the definition's
    if op == "prologue":
        T, H, HK, D, dims = case["T"], case["H"], case["HK"], case["D"], case["dims"]
        half = dims // 2
        i = torch.arange(half, device=DEV)
        # the pair i of a head: its two columns
        first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
        table = case["scale"] * torch.pow(torch.tensor(case["base"], dtype=f64, device=DEV),
                                          -2.0 * i.to(f64) / dims)
        z = torch.polar(torch.ones((T, half), dtype=f64, device=DEV),
                        torch.outer(st["positions"].to(f64), table))[:, None, :]

        def turned(x, norm, heads):
            y = x.to(f64).view(T, heads, D).clone()
            y /= torch.sqrt(y.pow(2).sum(-1, keepdim=True) / D + EPS)
            y *= norm.to(f64)
            c = torch.complex(y[..., first], y[..., second]) * z
            y[..., first], y[..., second] = c.real, c.imag
            return y

        k, v = st["k_pages"].to(f64), st["v_pages"].to(f64)
        flat = [c.transpose(1, 2).reshape(-1, HK, D) for c in (k, v)]
        flat[0][st["slots"].long()] = turned(st["k"], st["k_norm"], HK)
        flat[1][st["slots"].long()] = st["v"].to(f64).view(T, HK, D)
        k, v = (f.reshape(-1, case["page"], HK, D).transpose(1, 2).contiguous() for f in flat)
        return {"q": turned(st["q"], st["q_norm"], H), "k_pages": k, "v_pages": v}
    if op == "attention":
        H, HK, D = case["H"], case["HK"], case["D"]
        G = H // HK
        out = torch.zeros(st["q"].shape, dtype=f64, device=DEV)
        cu, kv = st["cu"].tolist(), st["kv"].tolist()
        for r, n in enumerate(kv):
            a, b = cu[r], cu[r + 1]
            pages = st["table"][r, :_pages(n, case["page"])].long()
            last = n - (b - a)  # the first new token's position
            for h in range(HK):
                k = st["k"][pages, h].reshape(-1, D)[:n].to(f64)
                v = st["v"][pages, h].reshape(-1, D)[:n].to(f64)
                hide = torch.ones((b - a, n), dtype=torch.bool, device=DEV).triu(last + 1)
                for g in range(h * G, h * G + G):
                    s = st["q"][a:b, g].to(f64) @ k.T * st["scale"]
                    s[hide] = -math.inf
                    out[a:b, g] = torch.softmax(s, -1) @ v
        return out
    x = st["x"]
    rows, V = x.shape
    k = case["top"]
    lp = torch.empty(rows, dtype=f64, device=DEV)
    ent, top = torch.empty_like(lp), torch.empty((rows, k), dtype=f64, device=DEV)
    for a in range(0, rows, 128):  # in parts: 64-bit rows of a large vocabulary
        y = torch.log_softmax(x[a:a + 128].to(f64), -1)
        lp[a:a + 128] = y.gather(1, st["tokens"][a:a + 128, None])[:, 0]
        ent[a:a + 128] = -torch.where(y.exp() > 0, y.exp() * y, 0.0).sum(-1)
        top[a:a + 128] = torch.topk(y, k, -1).values
    out = {"logprobs": lp, "entropy": ent}
    if k:
        out["top_ids"], out["top_logprobs"] = None, top
    return out
