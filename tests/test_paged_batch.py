"""What a paged batch keeps between steps (the plans themselves are made by a
stand-in on the CPU)."""

from __future__ import annotations

import dataclasses

import pytest

torch = pytest.importorskip("torch")
from autotuner_runtime import ops  # noqa: E402
from workloads import qwen3  # noqa: E402

CFG = dataclasses.replace(qwen3.Qwen3Config(), hidden_size=512, num_attention_heads=8,
                          num_key_value_heads=2, head_dim=64)


@pytest.fixture
def steps(monkeypatch):
    """(batch, step(rows), capturing(on)); a step's plan notes its number in cu_q."""
    state = {"on": False, "n": 0}

    def plan(table, lens, q_lens, free, count, page, T, out=None):
        R = lens.shape[0]
        out = out or ops.PagedPlan(*(torch.zeros(n, dtype=torch.int32) for n in (R + 1, R, T, T, 1, 1)))
        state["n"] += 1
        out.cu_q.fill_(state["n"])
        return out

    monkeypatch.setattr(ops, "paged_plan", plan)
    monkeypatch.setattr(qwen3, "_capturing", lambda t: state["on"], raising=False)
    batch = qwen3.PagedBatch(CFG, 1, 2, 4, 16, 64, "cpu")
    q = torch.zeros(2, dtype=torch.int32)
    return batch, lambda rows: batch.step(q, rows), lambda on: state.update(on=on)


def kept(batch) -> int:
    """Plans that the batch holds, wherever it does."""
    seen = set()

    def walk(v):
        if isinstance(v, ops.PagedPlan):
            seen.add(v.positions.data_ptr())
        elif isinstance(v, dict):
            for x in v.values():
                walk(x)
        elif isinstance(v, (list, tuple)):
            for x in v:
                walk(x)

    walk(vars(batch))
    return len(seen)


def test_steps_of_all_sizes_leave_few_plans(steps):
    batch, step, _ = steps
    for rows in range(1, 3000):
        step(rows)
    assert kept(batch) <= 65


def test_a_plan_stays_for_steps_of_as_many_rows(steps):
    batch, step, _ = steps
    a, b = step(3), step(40)
    assert a.cu_q.tolist() == [1, 1, 1] and b.cu_q.tolist() == [2, 2, 2]
    for _ in range(100):  # decoding between prompts of ever other sizes
        assert step(3) is a
        step(100 + int(a.cu_q[0]))
    old = step(40)
    n = int(old.cu_q[0])
    for rows in range(1000, 1200):
        step(rows)
    assert int(old.cu_q[0]) == n  # whoever holds a plan that the batch dropped, keeps it


def test_captured_plans_stay(steps):
    """Of a step that a capture holds, and of one whose plan a capture reads."""
    batch, step, capturing = steps
    capturing(True)
    a = step(3)
    capturing(False)
    b = step(7)
    capturing(True)
    assert batch.plan is b
    capturing(False)
    for rows in range(100, 400):
        step(rows)
    assert step(3) is a and batch.plan is a
    assert step(7) is b and batch.plan is b
    assert kept(batch) <= 67


def test_a_refused_call_changes_nothing(steps, monkeypatch):
    batch, step, _ = steps
    a = step(3)
    with monkeypatch.context() as m:
        def refuse(*args, **kw):
            raise ValueError("no")
        m.setattr(ops, "paged_plan", refuse)
        with pytest.raises(ValueError):
            step(3)
    assert batch.plan is a and step(3) is a


@pytest.mark.gpu
def test_graph_of_layers_after_steps_of_many_sizes():
    """A forward pass captured over a plan that was made before it, replayed after
    steps of more row counts than are kept."""
    from autotuner_runtime import hip

    cfg = dataclasses.replace(CFG, intermediate_size=1024, vocab_size=1000)
    model = qwen3.build(cfg, seed=3, num_layers=2)
    ids = [qwen3.tokens(90 + i, 3, cfg.vocab_size)[0] for i in range(6)]

    def run(between, forward):
        batch = model.make_batch(3, 60, page_size=16, max_len=320)
        prompts = torch.cat([qwen3.tokens(50 + i, n, cfg.vocab_size)[0] for i, n in enumerate((30, 15, 1))])
        batch.step(torch.tensor([30, 15, 1], dtype=torch.int32, device="cuda"), 46)
        model.forward_paged(prompts, batch)
        one, none = (torch.full((3,), v, dtype=torch.int32, device="cuda") for v in (1, 0))
        out = []
        for i, t in enumerate(ids):
            for rows in range(between):  # steps that bring nothing, in buffers of other sizes
                batch.step(none, 100 + rows + between * i)
            batch.step(one, 3, 1)
            out.append(forward(t, batch).clone())
        return out, batch.lens.tolist()

    want = run(0, model.forward_paged)
    graph, static, logits = torch.cuda.CUDAGraph(), ids[0].clone(), []

    def replay(t, batch):
        static.copy_(t)
        if not logits:
            torch.cuda.synchronize()
            with hip.graph_workspaces(), torch.cuda.graph(graph):
                logits.append(model.forward_paged(static, batch))
        graph.replay()
        return logits[0]

    got = run(70, replay)
    assert got[1] == want[1] == [36, 21, 7]
    assert all(torch.equal(a, b) for a, b in zip(got[0], want[0]))
