"""What a beam search refuses, before it takes anything."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from workloads import qwen3  # noqa: E402
from test_beams_model_gpu import CFG, batch_of, prompts, small  # noqa: E402


def test_refusals_take_no_pages():
    """What the selection would refuse behind the prompts' step."""
    model, ps = small(), prompts(20)
    for B, eos in ((65, None), (2, CFG.vocab_size), (2, -1)):
        batch = batch_of(model, 1, B)
        with pytest.raises(ValueError):
            qwen3.generate_beams(model, batch, ps, 3, eos)
        assert not batch.lens.any() and int(batch.free_count) == 200
