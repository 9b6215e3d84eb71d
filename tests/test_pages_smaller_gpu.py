"""Pools that are cut behind a compaction."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from workloads import qwen3  # noqa: E402
from test_beams_model_gpu import consistent, prompts, small  # noqa: E402


def test_requests_go_on_in_smaller_pools():
    """Half of the requests finish, the pools keep what the rest hold and two pages more;
    the next steps' logits are those of the batch that was not cut, and the pages run out
    where there are no more."""
    model, ps = small(), prompts(100, 37, 150, 5)
    lens = torch.tensor([p.numel() for p in ps], dtype=torch.int32, device="cuda")

    def start():
        batch = model.make_batch(4, 60, page_size=16, max_len=320)
        batch.step(lens, int(lens.sum()), 150)
        model.forward_paged(torch.cat(ps), batch)
        batch.finish(0)
        batch.finish(2)
        return batch

    whole, batch = start(), start()
    held = int(batch.compact())
    assert held == 4 and {p for r in (1, 3) for p in batch.block_table[r, :3 if r == 1 else 1].tolist()} \
        == set(range(4))
    P = held + 2
    for c in batch.caches:
        c.keys, c.values = c.keys[:P].clone(), c.values[:P].clone()
    batch.free_pages, batch.free_count = batch.free_pages[60 - P:], batch.free_count - (60 - P)
    consistent(batch, P)
    one = torch.tensor([0, 1, 0, 1], dtype=torch.int32, device="cuda")
    for i in range(12):
        ids = qwen3.tokens(70 + i, 2, 1000)[0]
        refused = batch.step(one, 2, 1).refused
        whole.step(one, 2, 1)
        assert int(refused) == 0
        a, b = model.forward_paged(ids, batch), model.forward_paged(ids, whole)
        assert torch.equal(a[[1, 3]], b[[1, 3]]), i
    consistent(batch, P)
    assert batch.lens.tolist() == [0, 49, 0, 17] and int(batch.free_count) == 0
    batch.finish(1)
    consistent(batch, P)
    assert int(batch.free_count) == 4
    refused = ops.paged_fork(batch.block_table, batch.lens, one * 3, batch.free_pages,
                             batch.free_count, batch.pools())
    assert int(refused) == 0
