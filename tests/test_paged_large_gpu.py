"""Paged attention of large steps: a long decoding request beside tens of thousands
of prompt tokens, and thousands of decoding requests."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from test_paged_gpu import BF, attention_64, check_attention, i32  # noqa: E402


@pytest.mark.parametrize("kv,n_q,H,HK,D,hint", [
    ([219] * 150 + [30000] + [219] * 151, [219] * 150 + [1] + [219] * 151, 64, 32, 64, None),
    ([30000] + [70] * 2500, [1] * 2501, 32, 32, 64, 1),
    ([70] * 4000 + [9000, 60], [1] * 4002, 32, 8, 128, 1),
])
def test_large_steps(kv, n_q, H, HK, D, hint):
    g = torch.Generator(device="cuda")
    g.manual_seed(len(kv))
    page, T, R = 16, sum(n_q), len(kv)
    W = -(-max(kv) // page)
    counts = [-(-n // page) for n in kv]
    P = sum(counts)
    kp, vp = (torch.randn((P, HK, page, D), generator=g, device="cuda").to(BF) for _ in range(2))
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    table = torch.full((R, W), -1, dtype=torch.int32, device="cuda")
    at, starts = 0, [0]
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
        starts.append(starts[-1] + n_q[r])
    q = torch.randn((T, H, D), generator=g, device="cuda").to(BF)
    out = ops.paged_attention(q, kp, vp, table, i32(starts), i32(kv), D ** -0.5, hint)
    long = kv.index(max(kv))
    for r in (0, 1, long, long + 1, R // 2, R - 1):
        ids = table[r, :counts[r]].long()
        k, v = (p[ids].transpose(1, 2).reshape(-1, HK, D)[:kv[r]].cpu() for p in (kp, vp))
        rows = slice(starts[r], starts[r + 1])
        check_attention(out[rows], *attention_64(q[rows], [k], [v], [n_q[r]], D ** -0.5), BF)
