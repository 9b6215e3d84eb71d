"""Beams that have ended take no part in a search's steps: no pages, no length, no rows."""

from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from workloads import qwen3  # noqa: E402
from test_beams_model_gpu import batch_of, consistent, prompts, small  # noqa: E402


def test_a_beam_that_ends_grows_no_longer():
    """One beam a prompt: the first comes to its eos as its second token at the latest, and
    20 tokens would pass the table's 96 keys. The pool holds eight pages of 16: six for its
    90 keys and one token, two for the other's 7 and 19."""
    model, ps = small(), prompts(90, 7)
    free = qwen3.generate_beams(model, batch_of(model, 2, 1), ps, 2)
    eos = int(free.sequences[0, 0, 1])
    first = free.sequences[0, 0].tolist()
    batch = batch_of(model, 2, 1, pages=8, max_len=96)
    got = qwen3.generate_beams(model, batch, ps, 20, eos)
    at = first.index(eos)
    assert got.sequences[0, 0].tolist() == first[:at + 1] + [eos] * (19 - at)
    assert got.finished[0, 0]
    consistent(batch, 8)
    assert int(batch.lens[0]) == 0
    if not got.finished[1, 0]:
        assert int(batch.lens[1]) == 7 + 19


@pytest.mark.parametrize("regions", [False, True])
def test_the_others_go_on_as_they_would(regions):
    """Prompts whose beams end at different steps: every sequence's score is the model's
    over it alone, up to its eos; the requests that are left hold what is alive."""
    model, ps, n, B = small(), prompts(130, 20, 45), 7, 4
    if regions:
        qwen3.install_regions(model)
    free = qwen3.generate_beams(model, batch_of(model, 3, B), ps, n)
    eos = int(free.sequences[0, 0, 1])
    batch = batch_of(model, 3, B)
    got = qwen3.generate_beams(model, batch, ps, n, eos)
    assert got.finished[0].any() and not got.finished.all()
    consistent(batch, 200)
    model = small()
    for r, p in enumerate(ps):
        for b in range(B):
            ids, caches, score, bar = p[None], model.make_cache(300), 0.0, 0.0
            tokens = got.sequences[r, b].tolist()
            if eos in tokens:
                assert set(tokens[tokens.index(eos):]) == {eos}
                tokens = tokens[:tokens.index(eos) + 1]
            for t in tokens:
                logits = model(ids, caches)[0, -1].double()
                score += float(torch.log_softmax(logits, -1)[t])
                # (the logits agree to 3e-2 of the largest: two correct orders of rounding
                # through two bf16 layers and the head)
                bar += 2 * 3e-2 * float(logits.abs().max())
                ids = torch.tensor([[t]], device="cuda")
            assert abs(score - float(got.scores[r, b])) <= bar, (r, b)
    # of a request in the last step: nothing, or the prompt's keys and a token a step
    for r, p in enumerate(ps):
        assert set(batch.lens[r * B:(r + 1) * B].tolist()) <= {0, p.numel() + n - 1}
    ended = got.finished.view(-1).sum()
    assert int((batch.lens == 0).sum()) <= int(ended)


def test_all_have_ended():
    """Steps behind the last beam's end: no request holds anything, nothing is refused."""
    model, ps = small(), prompts(60, 60)
    ps[1] = ps[0]
    eos = int(qwen3.generate_beams(model, batch_of(model, 2, 1), ps, 1).sequences[0, 0, 0])
    batch = batch_of(model, 2, 1, pages=8, max_len=64)
    got = qwen3.generate_beams(model, batch, ps, 30, eos)
    assert got.finished.all() and (got.sequences == eos).all()
    assert not batch.lens.any() and int(batch.free_count) == 8


def test_beams_without_a_continuation(monkeypatch):
    """Beams of score -inf (fewer candidates than beams, say) bring no tokens either, with
    no eos at all."""
    model, ps, B = small(), prompts(40, 30), 3
    choose, widths = ops.beam_select, []

    def fewer(logits, scores, **kw):
        s = choose(logits, scores, **kw)
        s.scores[0, 1:] = -math.inf
        s.parents[0, 1:], s.tokens[0, 1:] = 0, 0
        widths.append(batch.lens.tolist())
        return s

    monkeypatch.setattr(ops, "beam_select", fewer)
    batch = batch_of(model, 2, B)
    got = qwen3.generate_beams(model, batch, ps, 5)
    assert widths[-1] == [44, 0, 0, 34, 34, 34]
    assert (got.scores[0, 1:] == -math.inf).all() and got.scores[0, 0] > -math.inf
    consistent(batch, 200)
    monkeypatch.undo()
    alone = qwen3.generate_beams(model, batch_of(model, 1, B), ps[1:], 5)
    assert torch.equal(got.sequences[1], alone.sequences[0])
