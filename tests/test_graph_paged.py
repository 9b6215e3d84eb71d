"""Graph delivery of layers over a paged cache: what a graph reads beside the pools
(block table, plan, angles) is the batch's, and no other batch replays it."""

from __future__ import annotations

import dataclasses

import pytest

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from autotuner_runtime.graph import GraphWrapper, signature  # noqa: E402
from workloads import qwen3  # noqa: E402

CFG = dataclasses.replace(qwen3.Qwen3Config(), hidden_size=512, num_attention_heads=8,
                          num_key_value_heads=2, head_dim=64, intermediate_size=1024,
                          vocab_size=1000)


@pytest.fixture
def plans(monkeypatch):
    """``ops.paged_plan`` on the CPU: fresh arrays of a plan's shapes, or the given ones."""
    def plan(table, lens, q_lens, free, count, page, T, out=None):
        R = lens.shape[0]
        return out or ops.PagedPlan(*(torch.zeros(n, dtype=torch.int32) for n in (R + 1, R, T, T, 1, 1)))

    monkeypatch.setattr(ops, "paged_plan", plan)


def batch_over(pools=None):
    b = qwen3.PagedBatch(CFG, 1, 2, 4, 16, 64, "cpu")
    if pools is not None:
        b.caches[0].keys, b.caches[0].values = pools.caches[0].keys, pools.caches[0].values
    return b


def test_signatures_tell_batches_apart(plans):
    """Two batches over the same pools (as of a batch made where a freed one's pools
    lay), each given as a layer's cache and by itself."""
    a = batch_over()
    b = batch_over(a)
    x, q = torch.zeros(1, 3, 8), torch.zeros(2, dtype=torch.int32)
    for batch in (a, b):
        batch.step(q, 3)
    assert signature((x, a.caches[0])) != signature((x, b.caches[0]))
    assert signature((x, a)) != signature((x, b))
    before = signature((x, a.caches[0])), signature((x, a))
    a.step(q, 3)
    assert (signature((x, a.caches[0])), signature((x, a))) == before  # the same buffers again


def test_signatures_tell_plans_apart(plans):
    """Plans of one batch that lie in different places."""
    a = batch_over()
    x, q = torch.zeros(1, 3, 8), torch.zeros(2, dtype=torch.int32)
    a.step(q, 3)
    before = signature((x, a.caches[0]))
    a.step(q, 5)
    assert signature((x, a.caches[0])) != before


@pytest.mark.gpu
def test_layers_serve_a_second_batch_over_the_same_pools():
    model = qwen3.build(CFG, seed=3, num_layers=2)
    ps = [qwen3.tokens(50 + i, n, CFG.vocab_size)[0] for i, n in enumerate((30, 15, 1))]
    want, _ = qwen3.generate_paged(model, model.make_batch(3, 12, page_size=16, max_len=96), ps, 5)
    model.model.layers = torch.nn.ModuleList(GraphWrapper(layer) for layer in model.model.layers)
    first = model.make_batch(3, 12, page_size=16, max_len=96)
    got, _ = qwen3.generate_paged(model, first, ps, 5)
    assert torch.equal(got, want)
    second = model.make_batch(3, 12, page_size=16, max_len=96)
    second.free_pages.copy_(second.free_pages.flip(0))  # other pages for every request
    for c, d in zip(second.caches, first.caches):
        c.keys, c.values = d.keys, d.values
    ps = [p.flip(0) for p in ps]
    model.model.layers, kept = torch.nn.ModuleList(w.wrapped for w in model.model.layers), model.model.layers
    want, _ = qwen3.generate_paged(model, model.make_batch(3, 12, page_size=16, max_len=96), ps, 5)
    model.model.layers = kept
    got, _ = qwen3.generate_paged(model, second, ps, 5)
    assert torch.equal(got, want)
