"""The operators of a step over a paged cache against plain 64-bit forms: the
plan, the prologue, the attention, and the three in a row."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import hip, ops  # noqa: E402

DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16
I32 = torch.int32


def half_step(dt) -> float:
    return torch.finfo(dt).eps / 2


def i32(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def rnd(gen, *shape, dtype=BF):
    return torch.randn(shape, generator=gen).to(dtype).to(DEV)


def gen_of(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------------------
# the plan


def plan_by_hand(table, kv, q, free, count, page, T):
    """The definition, request after request."""
    table = [list(r) for r in table]
    W = len(table[0])
    cu, after, positions, slots = [0], [], [0] * T, [-1] * T
    end = taken = refused = 0
    for r, (n, m) in enumerate(zip(kv, q)):
        old, new = -(-n // page), -(-(n + m) // page)
        need = new - old if new <= W else 0
        first = end
        end += need
        ok = new <= W and (need == 0 or end <= count)
        if ok and need:
            taken = end
            for i in range(need):
                table[r][old + i] = free[count - 1 - (first + i)]
        refused += not ok
        for i in range(m):
            t, pos = cu[-1] + i, n + i
            positions[t] = pos
            if ok:
                slots[t] = table[r][pos // page] * page + pos % page
        after.append(n + m if ok else 0)
        cu.append(cu[-1] + m)
    return table, cu, after, positions, slots, count - taken, refused


@pytest.mark.parametrize("R,page,kv_hi,q_hi,spare,short", [
    (1, 16, 0, 1, 0, 0), (1, 64, 700, 1, 3, 0), (3, 16, 50, 40, 0, 0), (64, 32, 500, 1, 0, 0),
    (65, 16, 90, 33, 5, 0), (256, 64, 300, 20, 0, 40), (257, 128, 1000, 3, 1000, 0),
    (300, 16, 40, 17, 9, 150), (1000, 256, 2000, 4, 0, 3), (4096, 16, 60, 2, 1, 500),
    (2, 16, 0, 3000, 7, 0),
])
def test_plan(R, page, kv_hi, q_hi, spare, short):
    """short: pages missing from the free list, so that the last requests that
    need any are refused. Requests without a new token, without a key, and one
    that would pass the table's width are among them."""
    rng = np.random.default_rng(R * 1000 + page)
    kv = rng.integers(0, kv_hi + 1, R).tolist()
    q = rng.integers(0, q_hi + 1, R).tolist()
    q[0] = max(q[0], 1)
    W = max(-(-(a + b) // page) for a, b in zip(kv, q))
    if R > 60:  # one request too long for the table
        W = max(1, W - 1)
        kv = [min(a, W * page) for a in kv]
    ids = rng.permutation(R * (W + 1) + 50).tolist()
    table = [[ids.pop() if w < -(-n // page) else -7 for w in range(W)] for n in kv]
    need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(kv, q))
    count = max(0, need - short)
    free = (ids * (1 + need // max(1, len(ids))))[:need + 5]
    T = sum(q) + spare
    want = plan_by_hand(table, kv, q, free, count, page, T)
    dt = i32(table)
    ins = [i32(kv), i32(q), i32(free), i32([count])]
    kept = [t.clone() for t in ins]
    p = ops.paged_plan(dt, *ins, page, T)
    got = [dt, p.cu_q, p.kv_lens, p.positions, p.slots, p.free_count, p.refused]
    for g, w, name in zip(got, want, ("table", "cu_q", "kv_lens", "positions", "slots", "free", "refused")):
        assert g.flatten().tolist() == torch.tensor(w).flatten().tolist(), name
    assert all(torch.equal(a, b) for a, b in zip(ins, kept))
    if short:
        assert int(p.refused) > 0
    again = ops.paged_plan(dt, *ins, page, T)  # the same step again: the same answer
    assert all(torch.equal(a, b) for a, b in zip(p, again)) and dt.tolist() == want[0]


def test_plan_into_an_earlier_one():
    table, free = i32([[0, 0], [0, 0]]), i32([7, 8, 9, 10])
    kv, count = i32([0, 0]), i32([4])
    a = ops.paged_plan(table, kv, i32([3, 17]), free, count, 16, 20)
    at = [t.data_ptr() for t in a]
    b = ops.paged_plan(table, i32([3, 17]), i32([20, 0]), free, i32([1]), 16, 20, out=a)
    assert [t.data_ptr() for t in b] == at and b.kv_lens.tolist() == [23, 17]
    assert b.cu_q.tolist() == [0, 20, 20] and int(b.free_count) == 0 and int(b.refused) == 0
    for bad in (dict(num_tokens=21), dict(kv_lens=b.kv_lens), dict(free_count=b.free_count)):
        kw = dict(block_table=table, kv_lens=kv, q_lens=i32([1, 1]), free_pages=free,
                  free_count=count, page_size=16, num_tokens=20, out=b)
        with pytest.raises(ValueError):
            ops.paged_plan(**{**kw, **bad})


def test_plan_of_more_tokens_than_rows():
    """A request whose tokens pass the rows takes no page; the next ones, neither."""
    table, free = i32([[0, 0]] * 4), i32([7, 8, 9, 10])
    p = ops.paged_plan(table, i32([0, 3, 20, 5]), i32([10, 20, 0, 1]), free, i32([4]), 16, 29)
    assert p.kv_lens.tolist() == [10, 0, 20, 0] and int(p.refused) == 2
    assert int(p.free_count) == 3 and table.tolist() == [[10, 0], [0, 0], [0, 0], [0, 0]]
    assert p.slots.tolist() == [160 + i for i in range(10)] + [-1] * 19


def test_plan_of_empty_requests():
    p = ops.paged_plan(i32([[5], [6]]), i32([0, 16]), i32([0, 0]), i32([]), i32([0]), 16, 0)
    assert p.cu_q.tolist() == [0, 0, 0] and p.kv_lens.tolist() == [0, 16]
    assert p.positions.numel() == 0 and int(p.refused) == 0 and int(p.free_count) == 0


# ---------------------------------------------------------------------------
# the prologue


def prologue_64(x, w, D, eps, table, positions, interleaved):
    """rms_norm * w and the rotation in float64, from the definition: ([T, h, D],
    the size of what each output was made of)."""
    T = x.shape[0]
    y = x.double().reshape(T, -1, D)
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    size = y.abs()
    half = table.shape[0]
    ang = positions.double()[:, None, None] * table
    c, s = torch.cos(ang), torch.sin(ang)
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out, big = y.clone(), size.clone()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
    big[..., a] = big[..., b] = size[..., a] + size[..., b]
    return out, big


def near(got, want, big, dt):
    """One rounding (half a step of the result) and the fp32 arithmetic before it:
    a sum of 128 squares (128 x 2^-24, halved by the root: 4e-6 relative), sine and
    cosine within 2e-6, a few fp32 roundings: 1e-5 of the parts' size. (Results
    under fp16's normal range are off by half its smallest step, 2^-25.)"""
    err = (got.double() - want).abs()
    tol = half_step(dt) * want.abs() + 1e-5 * big + 2.0 ** -25
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("T,H,HK,D,dims,interleaved,page,dtype,norm,far", [
    (1, 4, 2, 128, 128, False, 16, BF, True, 0),
    (1, 32, 8, 64, 64, False, 64, FP, True, 131071),
    (5, 5, 1, 128, 128, True, 16, FP, True, 100000),
    (37, 3, 3, 64, 32, False, 32, BF, True, 7),
    (37, 32, 8, 128, 64, True, 128, FP, True, 90000),
    (130, 8, 2, 128, 96, False, 256, FP, True, 50000),
    (3, 7, 1, 64, 8, True, 16, BF, True, 3),
    (9, 2, 1, 64, 0, False, 16, BF, True, 3),        # nothing turned
    (9, 4, 2, 128, 128, False, 64, FP, False, 1000),  # no norm
    (2100, 4, 1, 64, 64, True, 64, BF, True, 0),
])
def test_prologue(T, H, HK, D, dims, interleaved, page, dtype, norm, far):
    g = gen_of(T * 7 + D + dims)
    qkv = rnd(g, T, (H + 2 * HK) * D, dtype=dtype)
    q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + HK) * D], qkv[:, (H + HK) * D:]
    qn, kn = ((1 + 0.1 * torch.randn(D, generator=g)).to(dtype).to(DEV) for _ in range(2))
    if not norm:
        qn = kn = None
    n_pages = -(-T // page) + 2
    kp, vp = rnd(g, n_pages, HK, page, D, dtype=dtype), rnd(g, n_pages, HK, page, D, dtype=dtype)
    table = ops.rope_table(dims, 1e6, 0.5)
    pos = (far + torch.arange(T)).to(I32).to(DEV)
    slots = torch.randperm(n_pages * page, generator=g)[:T].to(I32).to(DEV)
    if T > 4:  # tokens without a slot write nothing
        slots[1], slots[3] = -1, n_pages * page
    want_k, want_v = kp.clone(), vp.clone()
    out = ops.norm_rope_paged(q, k, v, qn, kn, H, HK, 1e-6, table, pos, slots, kp, vp,
                              traditional=interleaved)
    assert out.shape == (T, H, D) and out.dtype == dtype
    near(out, *prologue_64(q, qn, D, 1e-6, table, pos, interleaved), dtype)
    kept = (slots >= 0) & (slots < n_pages * page)
    at = slots[kept].long()
    yk, big = prologue_64(k, kn, D, 1e-6, table, pos, interleaved)
    near(kp[at // page, :, at % page], yk[kept], big[kept], dtype)
    assert torch.equal(vp[at // page, :, at % page], v.reshape(T, HK, D)[kept])
    # every other row as it was
    kp[at // page, :, at % page] = want_k[at // page, :, at % page]
    vp[at // page, :, at % page] = want_v[at // page, :, at % page]
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


def test_prologue_layouts():
    """Rows that are not 16-byte aligned, transposed rows, and rows repeated by a
    stride of zero give what contiguous ones do."""
    g = gen_of(3)
    T, H, HK, D = 6, 4, 2, 64
    flat = rnd(g, T * (H * D + 1) + 3)
    q = flat[3:3 + T * (H * D + 1)].view(T, H * D + 1)[:, :H * D]
    k = rnd(g, HK * D, T).t()
    v = rnd(g, 1, HK * D).expand(T, HK * D)
    table = ops.rope_table(D)
    pos, slots = i32(list(range(T))), i32(list(range(T)))
    got, want = [], []
    for dst, a, b, c in ((got, q, k, v), (want, q.contiguous(), k.contiguous(), v.contiguous())):
        kp, vp = torch.zeros(1, HK, 16, D, dtype=BF, device=DEV), torch.zeros(1, HK, 16, D, dtype=BF, device=DEV)
        dst += [ops.norm_rope_paged(a, b, c, None, None, H, HK, 1e-6, table, pos, slots, kp, vp), kp, vp]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# the attention


def make_cache(g, kv, page, HK, D, dtype, extra=2):
    """Pools in which the requests' pages lie scattered; what no key lies in is NaN."""
    counts = [-(-n // page) for n in kv]
    P = sum(counts) + extra
    order = torch.randperm(P, generator=g).tolist()
    W = max(1, max(counts)) + 1
    table = [[0] * W for _ in kv]
    kp = torch.full((P, HK, page, D), float("nan"), dtype=dtype)
    vp = kp.clone()
    ks, vs = [], []
    for r, n in enumerate(kv):
        k, v = (torch.randn((n, HK, D), generator=g).to(dtype) for _ in range(2))
        ks.append(k)
        vs.append(v)
        for w in range(counts[r]):
            table[r][w] = p = order.pop()
            m = min(page, n - w * page)
            kp[p, :, :m] = k[w * page:w * page + m].transpose(0, 1)
            vp[p, :, :m] = v[w * page:w * page + m].transpose(0, 1)
        for w in range(counts[r], W):
            table[r][w] = [-1, P + 3, 2 ** 31 - 1][w % 3]  # not a page: never needed
    return kp.to(DEV), vp.to(DEV), i32(table), ks, vs


def attention_64(q, ks, vs, n_q, scale):
    """(o, sum p |v| / sum p) [T, H, D] in float64, from the definition."""
    outs, sizes = [], []
    t = 0
    for k, v, n in zip(ks, vs, n_q):
        x = q[t:t + n].double().cpu()
        t += n
        H, HK, D = x.shape[1], k.shape[1], k.shape[2]
        L = k.shape[0]
        o = torch.zeros((n, H, D), dtype=torch.float64)
        a = torch.zeros_like(o)
        seen = torch.arange(L)[None, :] <= torch.arange(n)[:, None] + L - n
        for h in range(H):
            kk, vv = k[:, h // (H // HK)].double(), v[:, h // (H // HK)].double()
            s = (x[:, h] @ kk.T * scale).masked_fill(~seen, -np.inf)
            some = seen.any(1)
            p = torch.zeros_like(s)
            p[some] = torch.softmax(s[some], -1)
            o[:, h], a[:, h] = p @ vv, p @ vv.abs()
        outs.append(o)
        sizes.append(a)
    return torch.cat(outs), torch.cat(sizes)


def check_attention(got, want, size, dt):
    """Each probability is rounded to the type (half a step of it, so half a step of
    sum p |v| / sum p), the result once (half a step of itself); scores and sums are
    fp32: a score of 128 products errs by 128 x 2^-24 of the sum of their sizes
    (about 10 in log2 units here), 8e-5 of p, exponentials and sums by less: 2e-4."""
    err = (got.double().cpu() - want).abs()
    tol = half_step(dt) * (size + want.abs()) + 2e-4 * size + 2.0 ** -25
    assert bool((err <= tol).all()), float((err - tol).max())


def run_attention(kv, n_q, H, HK, D, page, dtype, scale=None, max_q_len=None, seed=0):
    g = gen_of(seed + sum(kv) + D + page)
    kp, vp, table, ks, vs = make_cache(g, kv, page, HK, D, dtype)
    T = sum(n_q)
    q = rnd(g, T, H, D, dtype=dtype)
    cu = i32([0] + np.cumsum(n_q).tolist())
    scale = D ** -0.5 if scale is None else scale
    out = ops.paged_attention(q, kp, vp, table, cu, i32(kv), scale, max_q_len)
    check_attention(out, *attention_64(q, ks, vs, n_q, scale), dtype)
    return out


@pytest.mark.parametrize("kv,n_q,H,HK,D,page,dtype", [
    ([1], [1], 8, 2, 128, 16, BF),                                   # one key
    ([16, 17, 31, 32, 33], [1] * 5, 8, 2, 64, 16, FP),               # pages' and tiles' ends
    ([127, 128, 129, 63, 1], [1] * 5, 32, 8, 128, 64, BF),
    ([700, 3, 1, 260, 511], [1] * 5, 10, 2, 128, 32, BF),            # 5 q heads a kv head
    ([0, 40, 0], [1, 1, 1], 4, 4, 64, 16, BF),                       # no keys: zeros
    ([5, 300], [5, 2], 8, 1, 64, 128, FP),                           # a prompt, two tokens
    ([100, 90, 80], [0, 3, 0], 8, 2, 128, 16, BF),                   # requests without tokens
    ([2500], [1], 32, 8, 128, 16, BF),
    ([9000], [1], 32, 8, 64, 256, FP),                               # past 64 tiles a wave
    ([1500, 20], [4, 4], 16, 2, 128, 64, FP),                        # 32 columns a request
    ([1500, 20], [5, 3], 64, 2, 64, 64, BF),                         # 160 columns: five blocks
    ([33], [33], 3, 3, 128, 16, BF),                                 # a prompt from nothing
    ([257, 64, 1000], [257, 1, 100], 8, 2, 128, 32, BF),             # mixed
    ([600], [600], 4, 1, 64, 16, FP),
    ([900, 700], [300, 700], 32, 8, 128, 64, BF),
    ([3, 2], [3, 2], 40, 1, 64, 16, BF),                             # 40 q heads on one kv head
    ([3, 40, 0], [5, 60, 70], 4, 2, 64, 16, BF),                     # more tokens than keys
    ([130, 300, 258], [4, 200, 3], 8, 2, 128, 64, BF),               # few tokens on both sides of a run's end
])
def test_attention(kv, n_q, H, HK, D, page, dtype):
    run_attention(kv, n_q, H, HK, D, page, dtype)


@pytest.mark.parametrize("scale", [-0.09, 0.0])
def test_attention_scales(scale):
    run_attention([200, 90], [1, 7], 8, 2, 128, 32, BF, scale=scale)


def test_attention_of_many_requests():
    """More requests than a wave has lanes, most of them short, some empty."""
    rng = np.random.default_rng(5)
    kv = rng.integers(1, 80, 333)
    n_q = np.minimum(rng.integers(0, 3, 333), kv)
    run_attention(kv.tolist(), n_q.tolist(), 4, 2, 64, 16, BF)


@pytest.mark.parametrize("R", [65, 193, 260])
def test_attention_of_many_requests_of_all_lengths(R):
    """Rows that are cut among rows that are not, prompts among single tokens, by
    64 requests a step and from a list of the work."""
    rng = np.random.default_rng(R)
    kv = rng.integers(1, 90, R)
    n_q = np.minimum(rng.integers(0, 3, R), kv)
    kv[[3, R // 2, R - 1]] = [2500, 700, 1301]
    n_q[[3, R // 2, R - 1]] = [1, 200, 33]
    kv[20], n_q[20] = 120, 120
    run_attention(kv.tolist(), n_q.tolist(), 8, 2, 64, 32, BF)
    run_attention(kv.tolist(), n_q.tolist(), 8, 2, 128, 16, FP, max_q_len=200)


@pytest.mark.parametrize("seed", range(6))
def test_attention_of_random_batches(seed):
    """Up to 64 requests: none, one, a few or hundreds of new tokens behind none,
    some or many keys, now and then more tokens than keys; wide blocks by length."""
    rng = np.random.default_rng(100 + seed)
    R = int(rng.integers(2, 65))
    kv = rng.choice([0, 1, 127, 128, 129, 256, 300, 640], R) + rng.integers(0, 40, R)
    n_q = np.minimum(rng.choice([0, 1, 2, 3, 8, 9, 33, 150], R), kv + (rng.random(R) < 0.1) * 5)
    G, HK = [(4, 2), (8, 1), (1, 4), (5, 2), (2, 2), (16, 1)][seed]
    kv[0], n_q[0] = [100, 4000][seed % 2], 60  # one in wide blocks at any of these
    n_q[1] = max(n_q[1], 1)
    D, page = [(64, 16), (128, 32)][seed // 3]
    run_attention(kv.tolist(), n_q.tolist(), G * HK, HK, D, page, [BF, FP][seed % 2])


def test_attention_without_a_workspace(monkeypatch):
    """The C entry without scratch: a workgroup a block, the same rows within
    rounding; scratch one byte short takes that path too."""
    kv, n_q = [3000, 10, 700], [1, 1, 90]
    want = run_attention(kv, n_q, 8, 2, 128, 64, BF)
    need = hip._paged_workspace_bytes
    for short in (lambda *a: 0, lambda *a: need(*a) - 1):
        monkeypatch.setattr(hip, "_paged_workspace_bytes", short)
        got = run_attention(kv, n_q, 8, 2, 128, 64, BF)
        assert float((got.float() - want.float()).abs().max()) < 0.05
    many = [50] * 300
    run_attention(many, [1] * 300, 4, 2, 64, 16, BF)


def test_attention_kernel_hint_changes_no_meaning():
    """max_q_len chooses kernels: too small, too large and absent give the rows."""
    for hint in (1, 7, 500, None):
        run_attention([400, 33, 260], [130, 1, 40], 8, 2, 64, 32, BF, max_q_len=hint)


def test_attention_beside_values_that_are_not_finite():
    """A prompt's last values are not finite: rows whose last key lies 96 keys or
    more before them, and other requests, do not know. Nor does decode of keys
    behind which such values lie in the page."""
    g = gen_of(34)
    kv, n_q = [300, 90, 33], [300, 1, 33]
    kp, vp, table, ks, vs = make_cache(g, kv, 16, 2, 64, BF)
    q, cu = rnd(g, sum(n_q), 8, 64), i32([0, 300, 301, 334])
    want, size = attention_64(q, ks, vs, n_q, 0.125)
    for bad in (float("nan"), float("inf")):
        vp[table[0, 299 // 16], :, 299 % 16] = bad
        kp[table[0, 299 // 16], :, 299 % 16] = bad
        out = ops.paged_attention(q, kp, vp, table, cu, i32(kv), 0.125)
        keep = torch.cat([torch.arange(300 - 96), torch.arange(300, 334)])
        check_attention(out[keep.to(DEV)], want[keep], size[keep], BF)


@pytest.mark.parametrize("R", [3, 200])
def test_attention_of_offsets_that_fall(R):
    """Of long rows nothing is written, and the workspace serves the next call as
    before."""
    g = gen_of(35 + R)
    kv, n_q = [700] * R, [1] * R
    kp, vp, table, ks, vs = make_cache(g, kv, 16, 1, 64, BF)
    q, lens = rnd(g, R, 4, 64), i32(kv)
    good = i32(list(range(R + 1)))
    want = ops.paged_attention(q, kp, vp, table, good, lens, 0.125, 1)
    check_attention(want, *attention_64(q, ks, vs, n_q, 0.125), BF)
    falling = i32([0, R] * R)[:R + 1]
    mark = torch.full_like(q, 7.0)
    hip.paged_attention(q, kp, vp, mark, table, falling, lens, 0.125)
    assert bool((mark == 7).all())
    assert torch.equal(ops.paged_attention(q, kp, vp, table, good, lens, 0.125, 1), want)


def test_attention_of_a_misaligned_query():
    g = gen_of(33)
    kp, vp, table, ks, vs = make_cache(g, [70], 16, 2, 64, BF)
    flat = rnd(g, 4 * 64 + 3)
    q = flat[3:].view(1, 4, 64)
    out = ops.paged_attention(q, kp, vp, table, i32([0, 1]), i32([70]), 0.125)
    check_attention(out, *attention_64(q, ks, vs, [1], 0.125), BF)


def test_attention_on_streams_and_threads():
    """Two streams and two threads at once, each with scratch of its own."""
    import threading

    g = gen_of(31)
    kv, n_q = [2900, 500], [1, 1]
    kp, vp, table, ks, vs = make_cache(g, kv, 64, 4, 128, BF)
    qs = [rnd(g, 2, 16, 128) for _ in range(4)]
    cu, lens = i32([0, 1, 2]), i32(kv)
    want = [ops.paged_attention(q, kp, vp, table, cu, lens, 0.1, 1) for q in qs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = ops.paged_attention(qs[i], kp, vp, table, cu, lens, 0.1, 1)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_in_graphs_at_other_lengths():
    """Two graphs of one shape, captured in scopes of their own and replayed in
    turn and at once, at lengths that change between replays."""
    g = gen_of(32)
    kv = [3000, 700]
    kp, vp, table, ks, vs = make_cache(g, kv, 64, 2, 64, BF)
    q = rnd(g, 2, 8, 64)
    cu, lens = i32([0, 1, 2]), i32(kv)
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    ops.paged_attention(q, kp, vp, table, cu, lens, 0.125, 1)
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with hip.graph_workspaces(), torch.cuda.graph(graph):
            outs.append(ops.paged_attention(q, kp, vp, table, cu, lens, 0.125, 1))
        graphs.append(graph)
    for now in ([3000, 700], [100, 1], [2049, 640], [3000, 700]):
        lens.copy_(i32(now))
        want = ops.paged_attention(q, kp, vp, table, cu, lens, 0.125, 1)
        check_attention(want, *attention_64(q, [k[:n] for k, n in zip(ks, now)],
                                            [v[:n] for v, n in zip(vs, now)], [1, 1], 0.125), BF)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_attention_leaves_rows_behind_the_last_request():
    """Rows of the token buffer that no request has are not written, and a cu_q
    that passes the buffer is held to it."""
    g = gen_of(11)
    kv, n_q = [50, 20], [1, 2]
    kp, vp, table, ks, vs = make_cache(g, kv, 16, 2, 64, BF)
    q = rnd(g, 6, 4, 64)
    out = torch.full_like(q, 7.0)
    cu = i32([0, 1, 3])
    hip.paged_attention(q, kp, vp, out, table, cu, i32(kv), 0.125)
    check_attention(out[:3], *attention_64(q[:3], ks, vs, n_q, 0.125), BF)
    assert bool((out[3:] == 7.0).all())
    # the last request's tokens pass the buffer: those that are in it are served
    # as the first of as many as are in it
    out2 = torch.full_like(q[:2], 7.0)
    hip.paged_attention(q[:2].contiguous(), kp, vp, out2, table, cu, i32(kv), 0.125)
    check_attention(out2, *attention_64(q[:2], ks, vs, [1, 1], 0.125), BF)


def test_attention_far_pages():
    """Pages past 2^32 bytes of a pool."""
    g = gen_of(12)
    page, HK, D = 256, 8, 128
    P = (1 << 32) // (page * HK * D * 2) + 3
    kp, vp = (torch.empty((P, HK, page, D), dtype=BF, device=DEV) for _ in range(2))
    n = 300
    ids = [P - 1, P - 2]
    ks, vs = [rnd(g, n, HK, D)], [rnd(g, n, HK, D)]
    for w, p in enumerate(ids):
        m = min(page, n - w * page)
        kp[p, :, :m] = ks[0][w * page:w * page + m].transpose(0, 1)
        vp[p, :, :m] = vs[0][w * page:w * page + m].transpose(0, 1)
    q = rnd(g, 1, 8, D)
    out = ops.paged_attention(q, kp, vp, i32([ids]), i32([0, 1]), i32([n]), D ** -0.5)
    check_attention(out, *attention_64(q, [ks[0].cpu()], [vs[0].cpu()], [1], D ** -0.5), BF)


def test_attention_repeats():
    """The same call gives the same bits."""
    a = run_attention([3000, 10, 700], [1, 1, 1], 32, 8, 128, 64, BF)
    b = run_attention([3000, 10, 700], [1, 1, 1], 32, 8, 128, 64, BF)
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# a step


def test_steps_in_a_row():
    """Prompts, then decode steps, then one more prompt beside them: plan, prologue
    and attention on one cache, against attention over all the keys so far. The
    pages come from the free list that each step leaves."""
    g = gen_of(21)
    H, HK, D, page, R, W = 8, 2, 64, 16, 3, 12
    P = R * W
    kp, vp = (torch.full((P, HK, page, D), float("nan"), dtype=BF, device=DEV) for _ in range(2))
    block, free = torch.zeros((R, W), dtype=I32, device=DEV), torch.randperm(P, generator=g).to(I32).to(DEV)
    count, lens = i32([P]), i32([0] * R)
    table = ops.rope_table(D, 1e4)
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(BF).to(DEV)
    seen = [([], []) for _ in range(R)]
    for n_q in ([20, 0, 33], [1, 0, 1], [1, 40, 1], [1, 1, 1], [2, 3, 1], [16, 1, 32]):
        T = sum(n_q) + 2  # two rows behind the last
        x = rnd(g, T, (H + 2 * HK) * D)
        q, k, v = x[:, :H * D], x[:, H * D:(H + HK) * D], x[:, (H + HK) * D:]
        p = ops.paged_plan(block, lens, i32(n_q), free, count, page, T)
        qr = ops.norm_rope_paged(q, k, v, w, w, H, HK, 1e-6, table, p.positions, p.slots, kp, vp)
        o = ops.paged_attention(qr, kp, vp, block, p.cu_q, p.kv_lens, D ** -0.5)
        # the keys as the cache holds them (the prologue's own test says how near they are)
        t, want, size = 0, [], []
        for r, n in enumerate(n_q):
            if n == 0:
                continue
            yk, big = prologue_64(k[t:t + n], w, D, 1e-6, table, p.positions[t:t + n], False)
            at = p.slots[t:t + n].long()
            got = kp[at // page, :, at % page]
            near(got, yk, big, BF)
            seen[r][0].append(got.cpu())
            seen[r][1].append(v[t:t + n].reshape(n, HK, D).cpu())
            a, b = attention_64(qr[t:t + n], [torch.cat(seen[r][0])], [torch.cat(seen[r][1])], [n], D ** -0.5)
            want.append(a)
            size.append(b)
            t += n
        check_attention(o[:t], torch.cat(want), torch.cat(size), BF)
        assert int(p.refused) == 0
        lens, count = p.kv_lens, p.free_count
    assert int(count) == P - sum(-(-int(n) // page) for n in lens)
