"""Requests of a paged batch that finish: pages back once, whatever the batch's size and
wherever its arrays lie."""

from __future__ import annotations

import dataclasses

import pytest

torch = pytest.importorskip("torch")
from workloads import qwen3  # noqa: E402

CFG = dataclasses.replace(qwen3.Qwen3Config(), hidden_size=128, num_attention_heads=2,
                          num_key_value_heads=1, head_dim=64)


def filled(layers, pages, device, beams=1):
    """Four requests: the first two hold three pages alike, and one more each."""
    b = qwen3.PagedBatch(CFG, layers, 4, pages, 16, 96, device, beams=beams)
    rows = [[7, 3, 9, 5], [7, 3, 9, 2], [1, 0, 0, 0], [8, 0, 0, 0]]
    b.block_table[:, :4] = torch.tensor(rows, dtype=torch.int32)
    b.lens.copy_(torch.tensor([50, 64, 1, 0], dtype=torch.int32))
    used = {7, 3, 9, 5, 2, 1}
    free = [i for i in range(pages if pages < 100 else 20) if i not in used]
    b.free_pages[:len(free)] = torch.tensor(free, dtype=torch.int32)
    b.free_count.fill_(len(free))
    return b, free


def check(b, free):
    def now():
        return b.free_pages[:int(b.free_count)].tolist()

    b.finish(3)  # holds nothing
    assert now() == free and b.lens.tolist() == [50, 64, 1, 0]
    b.finish(0)
    assert now() == free + [5] and b.lens.tolist() == [0, 64, 1, 0]
    b.finish(1)
    assert now() == free + [5, 2, 3, 7, 9] and b.lens.tolist() == [0, 0, 1, 0]
    b.finish(0)  # again
    b.finish(-2)
    assert now() == free + [5, 2, 3, 7, 9, 1] and not b.lens.any()
    with pytest.raises(IndexError):
        b.finish(4)


@pytest.mark.parametrize("layers", [0, 1])
def test_on_the_cpu(layers):
    check(*filled(layers, 12, "cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("layers,pages", [(0, 12), (1, 12), (1, (1 << 20) + 7)])
def test_on_the_gpu(layers, pages):
    """Among them more pages than a fork's bitmaps have bits."""
    check(*filled(layers, pages, "cuda"))


def test_beams_over_too_many_pages():
    """Refused when the batch is made, not at its first fork."""
    with pytest.raises(ValueError, match="pages"):
        qwen3.PagedBatch(CFG, 0, 4, (1 << 20) + 1, 16, 96, "cpu", beams=2)
    qwen3.PagedBatch(CFG, 0, 4, 1 << 20, 16, 96, "cpu", beams=2)
