"""Scratch with tickets, of several graphs captured in one scope: each graph zeroes
it before its own first use, whichever of them is replayed first."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
from autotuner_runtime import hip  # noqa: E402

CPU = torch.device("cpu")


@pytest.fixture
def capture(monkeypatch):
    """Makes the current stream count as capturing, by a capture's number."""
    state = {"id": None}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["id"] is not None)
    monkeypatch.setattr(hip, "_capture_id", lambda stream: state["id"], raising=False)
    return lambda number: state.update(id=number)


@pytest.mark.parametrize("zero,clear", [(64, 64), (True, 5000)])
def test_every_capture_of_a_scope_fills(capture, zero, clear):
    """As if what the fills' nodes did had not happened yet when the next graph is
    replayed: the bytes are dirty when each capture begins."""
    def take(n=5000):
        return hip._workspace("paged", CPU, 21, n, zero=zero)

    with hip.graph_workspaces():
        capture(1)
        a = take()
        assert not a[:clear].any()
        a.fill_(7)
        assert take() is a and bool((a == 7).all())   # one fill a capture
        capture(2)
        assert take(4000) is a and not a[:clear].any() and bool((a[clear:] == 7).all())
        a.fill_(7)
        assert take() is a and bool((a == 7).all())
        big = take(9000)                               # outgrown within a capture
        assert big is not a and not big[:clear].any()
        big.fill_(7)
        assert take(9000) is big and bool((big == 7).all())
        capture(3)
        assert take() is big and not big[:clear].any()


def test_no_fill_without_tickets(capture, monkeypatch):
    """... nor is the capture asked for where nothing has to be zero, or where no
    scope shares anything."""
    def refuse(stream):
        raise AssertionError("asked")

    monkeypatch.setattr(hip, "_capture_id", refuse)
    with hip.graph_workspaces():
        capture(1)
        a = hip._workspace("sdpa", CPU, 22, 5000)
        a.fill_(7)
        capture(2)
        assert hip._workspace("sdpa", CPU, 22, 5000) is a and bool((a == 7).all())
    assert not hip._workspace("paged", CPU, 22, 5000, zero=64)[:64].any()


def _cases():
    """(kind, call, a fresh input) of every entry with tickets, at sizes that use them."""
    from autotuner_runtime import ops

    g = torch.Generator(device="cuda")
    g.manual_seed(5)

    def rnd(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    kp, vp = rnd(50, 2, 64, 64), rnd(50, 2, 64, 64)
    table, cu, lens = i32([list(range(47)), [47, 48, 49] + [0] * 44]), i32([0, 1, 2]), i32([3000, 180])
    long_cu, long_lens = i32([0, 90, 91]), i32([3000, 180])
    tok = torch.zeros(3, dtype=torch.int64, device="cuda")
    w1, b1, w2, b2 = (rnd(*s, dtype=torch.float32) for s in ((2048, 1024), (2048,), (68, 2048), (68,)))
    return [
        ("decode", lambda q: ops.paged_attention(q, kp, vp, table, cu, lens, 0.125, 1), rnd(2, 8, 64)),
        ("prompt", lambda q: ops.paged_attention(q, kp, vp, table, long_cu, long_lens, 0.125),
         rnd(91, 8, 64)),
        ("logprobs", lambda x: ops.token_logprobs(x, tok, 5), rnd(3, 65537)),
        ("tiny mlp", lambda x: ops.gelu_mlp_f32(x, w1, b1, w2, b2), rnd(20, 1024, dtype=torch.float32)),
    ]


@pytest.mark.gpu
def test_second_graph_of_a_scope_replayed_first():
    """Three graphs captured in one scope over each entry, replayed in an order in
    which the first is last, then in turn with eager calls between."""
    for name, call, x in _cases():
        def parts(r):
            return list(r) if isinstance(r, tuple) else [r]

        call(x)  # (library and eager scratch, outside the captures)
        static = x.clone()
        torch.cuda.synchronize()
        graphs, outs = [], []
        with hip.graph_workspaces():
            for _ in range(3):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    outs.append(parts(call(static)))
                graphs.append(graph)
        for i in (2, 1, 2, 0, 1, 0, 2, 2):
            static.copy_(torch.roll(static, 1, dims=-1))
            want = parts(call(static))
            for o in outs[i]:
                o.zero_()
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want)), (name, i)


@pytest.mark.gpu
def test_captures_have_numbers():
    """One number a capture, on the streams that join it too; none outside."""
    x = torch.zeros(8, device="cuda")
    seen = []
    for _ in range(3):
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            here = torch.cuda.current_stream()
            ids = [hip._capture_id(here.cuda_stream)]
            x.add_(1)
            side.wait_stream(here)
            with torch.cuda.stream(side):
                ids.append(hip._capture_id(side.cuda_stream))
                x.add_(1)
            here.wait_stream(side)
            ids.append(hip._capture_id(here.cuda_stream))
        assert len(set(ids)) == 1
        seen.append(ids[0])
    assert len(set(seen)) == 3
    with pytest.raises(ValueError, match="not being captured"):
        hip._capture_id(torch.cuda.Stream().cuda_stream)
    x.add_(1)
    torch.cuda.synchronize()
