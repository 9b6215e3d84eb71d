"""Token log probabilities of logits far from zero: masks of large finite values
and references on both sides of where the sums change their units."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import hip  # noqa: E402
from test_logprobs_gpu import BF, DEV, F32, FP, check  # noqa: E402

FILLS = [-1e4, -6e4, -1e6, -1.1e6, -1e9, -1e10, -1e12, -1e15, -1e20, -1e25, -1e30, -3e38]


@pytest.fixture(params=["split", "row a workgroup"])
def scratch(request, monkeypatch):
    if request.param != "split":
        monkeypatch.setattr(hip, "_logprobs_workspace_bytes", lambda *a: 0)


@pytest.mark.parametrize("V", [3001, 151936])
@pytest.mark.parametrize("dtype,fill", [(d, f) for d in (BF, FP, F32) for f in FILLS
                                        if d is not FP or f >= -65504])
def test_masks_of_large_values(scratch, dtype, fill, V):
    """Real logits in the last chunk alone, in the first alone, in both; a row of
    the mask; masks of two sizes; the mask's negative among zeros."""
    x = torch.full((6, V), fill, dtype=dtype)
    real = torch.tensor([1.0, 2.5, 2.0, -3.0], dtype=dtype)
    x[0, V - 4:] = real
    x[1, :4] = real
    x[2, 7:11] = real
    x[2, V - 9:V - 5] = real + 40
    x[4, ::2] = fill / 2
    x[4, 1500] = 0.5
    x[5] = 0.0
    x[5, V // 2] = -fill
    x = x.to(DEV)
    r = check(x, torch.tensor([V - 3, 0, 3, V - 1, 1500, V // 2], device=DEV), 5)
    assert abs(float(r.entropy[3]) - math.log(V)) < 1e-5
    assert r.top_ids[3].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("centre", [2.0 ** 20, 2.0 ** 20 - 45, 1e5, 3e6, 1e8])
@pytest.mark.parametrize("sign", [1, -1])
def test_rows_around_a_large_value(scratch, centre, sign):
    """fp32 rows whose values spread by hundreds around a large one, ascending,
    descending and mixed: the reference moves across it many times."""
    V = 20000
    up = sign * centre + torch.linspace(-300, 300, V)
    g = torch.Generator()
    g.manual_seed(1)
    rows = [up, up.flip(0), up[torch.randperm(V, generator=g)],
            sign * centre + 20 * torch.randn(V, generator=g)]
    check(torch.stack(rows).to(DEV), torch.tensor([V - 1, 0, 17, 33], device=DEV), 9)
