"""Several requests through a Qwen3-shaped model over a paged cache: against one
request at a time over contiguous caches, with and without the regions, captured
in a graph, and with pages that run out."""

from __future__ import annotations

import dataclasses

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import hip, ops  # noqa: E402
from autotuner_runtime.graph import GraphWrapper  # noqa: E402
from workloads import qwen3  # noqa: E402

DEV = "cuda"
CFG = dataclasses.replace(qwen3.Qwen3Config(), hidden_size=512, num_attention_heads=8,
                          num_key_value_heads=2, head_dim=64, intermediate_size=1024,
                          vocab_size=1000)


def small(seed=3):
    return qwen3.build(CFG, seed=seed, num_layers=2)


def prompts(*lens):
    return [qwen3.tokens(50 + i, n, CFG.vocab_size)[0] for i, n in enumerate(lens)]


def close(a, b, bar=3e-2):
    """Two correct orders of rounding through two bf16 layers and the head (the
    contiguous prologue rounds three times where the paged one rounds once)."""
    err = float((a.float() - b.float()).abs().max() / b.float().abs().max())
    assert err <= bar, err


def test_requests_together_equal_each_alone():
    model, ps, n = small(), prompts(1, 20, 133, 64), 5
    batch = model.make_batch(len(ps), 24, page_size=16, max_len=160)
    tokens, lps = qwen3.generate_paged(model, batch, ps, n, top=3)
    assert tokens.shape == (n, len(ps))
    assert batch.lens.tolist() == [p.numel() + n - 1 for p in ps]
    used = sum(-(-(p.numel() + n - 1) // 16) for p in ps)
    assert int(batch.free_count) == 24 - used and int(batch.plan.refused) == 0
    # teacher-forced, one request at a time
    for r, p in enumerate(ps):
        caches = model.make_cache(200)
        ids = p[None]
        for i in range(n):
            logits = model(ids, caches)[0, -1].float()
            lp = torch.log_softmax(logits, -1)
            # the paged logits through what was reported of them: log softmax moves
            # by at most twice what the logits do
            bar = 2 * 3e-2 * float(logits.abs().max())
            assert abs(float(lps[i].logprobs[r] - lp[tokens[i, r].long()])) <= bar
            assert float((lps[i].top_logprobs[r] - lp[lps[i].top_ids[r].long()]).abs().max()) <= bar
            assert int(lps[i].top_ids[r, 0]) == int(tokens[i, r])
            assert float(lps[i].logprobs[r]) == float(lps[i].top_logprobs[r, 0])
            ids = tokens[i, r].long().view(1, 1)


def test_logits_match_and_regions_change_nothing():
    model, ps = small(), prompts(40, 7)
    lens = torch.tensor([40, 7], dtype=torch.int32, device=DEV)

    def prefill():
        batch = model.make_batch(2, 8, page_size=32, max_len=128)
        batch.step(lens, 47)
        return model.forward_paged(torch.cat(ps), batch), batch

    plain, b0 = prefill()
    for r, p in enumerate(ps):
        close(plain[r], model(p[None], model.make_cache(64))[0, -1])
    qwen3.install_regions(model)
    spliced, b1 = prefill()
    assert torch.equal(plain, spliced)
    for c0, c1 in zip(b0.caches, b1.caches):
        assert torch.equal(c0.keys, c1.keys) and torch.equal(c0.values, c1.values)


def test_decode_step_in_a_graph():
    """Plan, model, argmax and log probabilities of a decode step as one graph,
    replayed with eager work between; every replay against the eager step. Pages
    end inside the replays."""
    model, ps, n = small(), prompts(30, 15, 1), 6
    qwen3.install_regions(model)

    def start():
        batch = model.make_batch(3, 12, page_size=16, max_len=96)
        lens = [p.numel() for p in ps]
        batch.step(torch.tensor(lens, dtype=torch.int32, device=DEV), sum(lens))
        return batch, ops.argmax(model.forward_paged(torch.cat(ps), batch)).long()

    one = torch.ones(3, dtype=torch.int32, device=DEV)

    def decode(ids, batch):
        batch.step(one, 3, 1)
        logits = model.forward_paged(ids, batch)
        ids = ops.argmax(logits).long()
        return ids, logits, ops.token_logprobs(logits, ids, 4)

    batch, ids = start()
    eager = []
    for _ in range(n):
        ids, logits, lp = decode(ids, batch)
        eager.append((ids, logits, *lp))
    end = batch.lens.tolist()

    batch, first = start()
    static = first.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with hip.graph_workspaces(), torch.cuda.graph(graph):
        out, logits, lp = decode(static, batch)
    for i in range(n):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, logits, *lp), eager[i])), i
        torch.randn(1000, 1000, device=DEV) @ torch.randn(1000, 1000, device=DEV)
        static.copy_(out)
    assert batch.lens.tolist() == end


def test_generation_past_the_pages():
    """Two prompts of 20 and 30 tokens hold four pages of 16; a fourth
    new token's step needs a fifth, and a row of the table holds 32 tokens here."""
    model, ps = small(), prompts(20, 30)
    qwen3.generate_paged(model, model.make_batch(2, 4, page_size=16, max_len=96), ps, 3)
    for pages, max_len in ((4, 96), (3, 96), (8, 32)):
        with pytest.raises(RuntimeError, match="ran out"):
            qwen3.generate_paged(model, model.make_batch(2, pages, page_size=16,
                                                         max_len=max_len), ps, 6)
    batch = model.make_batch(2, 8, page_size=16, max_len=96)
    for bad, n in ((ps, 0), ([], 2), ([ps[0], ps[0][:0]], 2), (ps[:1], 2)):
        with pytest.raises(ValueError):
            qwen3.generate_paged(model, batch, bad, n)


def test_layers_in_graphs():
    """Each layer wrapped for graph delivery: captured at the first step of a shape
    and replayed at the following ones, whose plans say something else."""
    model, ps, n = small(), prompts(30, 15, 1), 5
    want_batch = model.make_batch(3, 12, page_size=16, max_len=96)
    want, _ = qwen3.generate_paged(model, want_batch, ps, n)
    layers = [GraphWrapper(layer) for layer in model.model.layers]
    model.model.layers = torch.nn.ModuleList(layers)
    for _ in range(2):
        batch = model.make_batch(3, 12, page_size=16, max_len=96)
        got, _ = qwen3.generate_paged(model, batch, ps, n)
        assert torch.equal(got, want)
        for a, b in zip(batch.caches, want_batch.caches):
            for r in range(3):
                m = int(batch.lens[r])
                for w in range(-(-m // 16)):
                    rows = min(16, m - 16 * w)
                    i, j = int(batch.block_table[r, w]), int(want_batch.block_table[r, w])
                    assert torch.equal(a.keys[i, :, :rows], b.keys[j, :, :rows])
    assert layers[0].stats["replays"] > layers[0].stats["captures"]


def test_pages_that_run_out_and_come_back():
    """A request that gets no pages keeps what it has and waits; its neighbours'
    logits are what they are without it; freed pages serve it."""
    model, ps = small(), prompts(30, 40, 20)
    ids = torch.cat(ps)
    batch = model.make_batch(3, 6, page_size=16, max_len=96)  # 2 + 3 + 2 pages wanted
    batch.step(torch.tensor([30, 40, 20], dtype=torch.int32, device=DEV), 90)
    got = model.forward_paged(ids, batch)
    assert int(batch.plan.refused) == 1 and batch.lens.tolist() == [30, 40, 0]
    assert int(batch.free_count) == 1
    roomy = model.make_batch(3, 9, page_size=16, max_len=96)
    roomy.step(torch.tensor([30, 40, 20], dtype=torch.int32, device=DEV), 90)
    want = model.forward_paged(ids, roomy)
    close(got[:2], want[:2])
    batch.finish(1)
    assert int(batch.free_count) == 4 and batch.lens.tolist() == [30, 0, 0]
    batch.step(torch.tensor([0, 0, 20], dtype=torch.int32, device=DEV), 20, 20)
    late = model.forward_paged(ps[2], batch)
    assert int(batch.plan.refused) == 0 and batch.lens.tolist() == [30, 0, 20]
    close(late[2], want[2])
    assert sorted(batch.free_pages[:int(batch.free_count)].tolist()
                  + batch.block_table[0, :2].tolist() + batch.block_table[2, :2].tolist()) == list(range(6))
