"""Small terms behind large ones in the sums of log probabilities."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import hip, ops  # noqa: E402
from test_logprobs_gpu import BF, DEV, F32, FP, reference  # noqa: E402


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_small_terms_behind_a_large_one(monkeypatch, dtype, split):
    """Every lane of a workgroup that has the row meets one logit of 0 first, then
    hundreds of -17: each e^-17 is under half a step of 1 in fp32, together they are
    2.4e-5 of the sum. A chunk's 16 values of a lane are added by themselves, then the
    chunk to what the lane has, the lanes and waves to each other: 16 + V / 4096 + 12
    roundings of 2^-24 in a row, and the 40 that exponentials and logarithm may err."""
    V, N = 151936, 4 if dtype is F32 else 8
    if not split:
        monkeypatch.setattr(hip, "_logprobs_workspace_bytes", lambda *a: 0)
    x = torch.full((2, V), -17.0, dtype=dtype)
    x[:, :4096].view(2, 4, -1, N)[:, :, :64, 0] = 0.0
    x = x.to(DEV)
    tok = torch.tensor([0, V - 1], device=DEV)
    lp, ent, _, _ = reference(x, tok, 1)
    r = ops.token_logprobs(x, tok)
    n = (16 + V / 4096 + 12 + 40) * 2.0 ** -24
    got = r.logprobs.cpu().numpy().astype(np.float64)
    assert (np.abs(got - lp) <= n + 2.0 ** -23 * np.abs(lp)).all(), np.abs(got - lp)
    e = r.entropy.cpu().numpy().astype(np.float64)
    assert (np.abs(e - ent) <= 3 * n * (1 + np.abs(ent))).all()
