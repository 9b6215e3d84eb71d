"""Beam search through a Qwen3-shaped model over a paged cache: selection, forked pages
and attention behind shared prefixes together."""

from __future__ import annotations

import dataclasses
import math

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


def batch_of(model, R, B, pages=200, page=16, max_len=400):
    return model.make_batch(R * B, pages, page_size=page, max_len=max_len, beams=B)


def pages_in_use(batch):
    used = set()
    for row, n in zip(batch.block_table.tolist(), batch.lens.tolist()):
        used |= set(row[:-(-n // batch.page_size)])
    return used


def consistent(batch, n_pages):
    """Every page is in use or free, once, and part-filled ones have one owner."""
    free = batch.free_pages.tolist()[:int(batch.free_count)]
    used = pages_in_use(batch)
    assert sorted(free + list(used)) == list(range(n_pages))
    last = [row[n // batch.page_size] for row, n in zip(batch.block_table.tolist(), batch.lens.tolist())
            if n % batch.page_size]
    assert len(set(last)) == len(last)


def test_beams_score_what_each_scores_alone():
    """Every sequence's score against the model run over it alone, on a contiguous cache.
    The logits agree to 3e-2 of the largest (two correct orders of rounding through two bf16
    layers and the head), so each token's log probability to twice that."""
    model, ps, n, B = small(), prompts(200, 37, 1), 6, 4
    batch = batch_of(model, 3, B)
    got = qwen3.generate_beams(model, batch, ps, n)
    assert got.sequences.shape == (3, B, n) and not got.finished.any()
    consistent(batch, 200)
    for r, p in enumerate(ps):
        assert len({tuple(s) for s in got.sequences[r].tolist()}) == B
        assert got.scores[r].tolist() == sorted(got.scores[r].tolist(), reverse=True)
        for b in range(B):
            ids, caches, score, bar = p[None], model.make_cache(300), 0.0, 0.0
            for t in got.sequences[r, b].tolist():
                logits = model(ids, caches)[0, -1].double()
                score += float(torch.log_softmax(logits, -1)[t])
                bar += 2 * 3e-2 * float(logits.abs().max())
                ids = torch.tensor([[t]], device=DEV)
            assert abs(score - float(got.scores[r, b])) <= bar, (r, b)
    for r in range(12):
        batch.finish(r)
    assert int(batch.free_count) == 200 and not batch.lens.any()


def test_one_beam_is_greedy():
    model, ps = small(), prompts(40, 7)
    want, lps = qwen3.generate_paged(model, model.make_batch(2, 20, page_size=16, max_len=96), ps, 8)
    got = qwen3.generate_beams(model, batch_of(model, 2, 1), ps, 8)
    assert torch.equal(got.sequences[:, 0].T, want)
    total = sum(lp.logprobs.double() for lp in lps)
    assert float((got.scores[:, 0].double() - total).abs().max()) < 8 * 2.0 ** -18


def test_sharing_changes_no_more_than_rounding():
    """The same search with every request's attention by itself: the scores, by the bound
    above over three tokens."""
    model, ps = small(), prompts(250, 160)
    a = qwen3.generate_beams(model, batch_of(model, 2, 5), ps, 3)
    batch = batch_of(model, 2, 5)
    batch.cu_groups = None
    b = qwen3.generate_beams(model, batch, ps, 3)
    largest = max(float(model(p[None], model.make_cache(300)).abs().max()) for p in ps)
    assert float((a.scores - b.scores).abs().max()) <= 3 * 2 * 3e-2 * largest


def test_beams_that_end():
    model, ps, n = small(), prompts(130, 20), 6
    free = qwen3.generate_beams(model, batch_of(model, 2, 4), ps, n)
    eos = int(free.sequences[0, 0, 2])  # a token that the best beam comes to
    batch = batch_of(model, 2, 4)
    got = qwen3.generate_beams(model, batch, ps, n, eos)
    consistent(batch, 200)
    ended = (got.sequences == eos).any(-1)
    assert torch.equal(got.finished, ended) and ended[0].any()
    for r in range(2):
        for b in range(4):
            s = got.sequences[r, b].tolist()
            if eos in s:
                assert set(s[s.index(eos):]) == {eos}
    assert (got.scores[:, :-1] >= got.scores[:, 1:]).all()


def test_regions_change_nothing():
    model, ps = small(), prompts(150, 33)
    want = qwen3.generate_beams(model, batch_of(model, 2, 3), ps, 4)
    qwen3.install_regions(model)
    got = qwen3.generate_beams(model, batch_of(model, 2, 3), ps, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def start(model, ps, B, pages=200):
    batch = batch_of(model, len(ps), B, pages)
    lens = torch.zeros(len(ps) * B, dtype=torch.int32, device=DEV)
    lens[::B] = torch.tensor([p.numel() for p in ps], dtype=torch.int32, device=DEV)
    batch.step(lens, sum(p.numel() for p in ps), max(p.numel() for p in ps))
    logits = model.forward_paged(torch.cat(ps), batch)
    scores = torch.full((len(ps), B), -math.inf, device=DEV)
    scores[:, 0] = 0.0
    s = ops.beam_select(logits, scores)
    assert int(batch.fork(s.parents.view(-1))) == 0
    return batch, s


def advance(model, batch, one, ids, scores, width):
    """One step of the search: plan, model, selection, fork."""
    batch.step(one, one.shape[0], 1)
    logits = model.forward_paged(ids, batch)
    s = ops.beam_select(logits, scores, width)
    batch.fork(s.parents.view(-1))
    return s, logits


@pytest.mark.parametrize("compact", [False, True])
def test_step_in_a_graph(compact):
    """A whole step as one graph, replayed with eager work between, against the eager
    one; with the pool compacted before every step, too."""
    model, ps, B, n = small(), prompts(140, 30, 3), 4, 6
    qwen3.install_regions(model)
    one = torch.ones(12, dtype=torch.int32, device=DEV)

    batch, s = start(model, ps, B)
    eager = []
    for _ in range(n):
        s, logits = advance(model, batch, one, s.tokens.view(-1).long(), s.scores, B)
        eager.append((*s, logits))
    end = batch.lens.tolist()

    batch, s = start(model, ps, B)
    ids, scores = s.tokens.view(-1).long(), s.scores.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with hip.graph_workspaces(), torch.cuda.graph(graph):
        if compact:
            batch.compact()
        out, logits = advance(model, batch, one, ids, scores, B)
    for i in range(n):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*out, logits), eager[i])), i
        consistent(batch, 200)
        torch.randn(1000, 1000, device=DEV) @ torch.randn(1000, 1000, device=DEV)
        ids.copy_(out.tokens.view(-1)), scores.copy_(out.scores)
    assert batch.lens.tolist() == end
    if compact:
        live = int(batch.compact())
        assert pages_in_use(batch) == set(range(live))


def test_layers_in_graphs():
    model, ps = small(), prompts(140, 15)
    want = qwen3.generate_beams(model, batch_of(model, 2, 3), ps, 5)
    layers = [GraphWrapper(layer) for layer in model.model.layers]
    model.model.layers = torch.nn.ModuleList(layers)
    for _ in range(2):
        got = qwen3.generate_beams(model, batch_of(model, 2, 3), ps, 5)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert layers[0].stats["replays"] > layers[0].stats["captures"]


def test_pages_that_run_out():
    """Two prompts of 20 tokens hold two pages each of 16, and three beams of each one more:
    eight pages; four more tokens fill none. With seven the first fork is refused."""
    model, ps = small(), prompts(20, 20)
    qwen3.generate_beams(model, batch_of(model, 2, 3, pages=8), ps, 4)
    for pages, max_len in ((7, 96), (200, 22)):
        with pytest.raises(RuntimeError, match="ran out"):
            qwen3.generate_beams(model, batch_of(model, 2, 3, pages, max_len=max_len), ps, 16)
    for bad, n in ((ps, 0), ([], 2), (ps[:1], 2), ([ps[0], ps[0][:0]], 2)):
        with pytest.raises(ValueError):
            qwen3.generate_beams(model, batch_of(model, 2, 3), bad, n)


def test_a_request_that_finishes_leaves_shared_pages():
    model, ps, B = small(), prompts(100), 3
    batch, s = start(model, ps, B)
    table = batch.block_table.tolist()
    assert table[0][:6] == table[1][:6] == table[2][:6]
    batch.finish(0)
    assert batch.lens.tolist() == [0, 100, 100]
    consistent(batch, 200)
    assert set(table[1][:6]) <= pages_in_use(batch)
    batch.finish(1)
    batch.finish(2)
    assert int(batch.free_count) == 200
