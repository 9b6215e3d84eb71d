"""How much scratch the paged attention asks for (no device needed): states for
blocks that can be cut, none for those that are not."""

from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")
from autotuner_runtime import hip  # noqa: E402

MB = 1 << 20


@pytest.fixture(scope="module")
def query():
    f = ctypes.CDLL(str(hip.library_path())).mi_paged_attention_workspace_bytes
    f.argtypes, f.restype = hip.SIGNATURES["mi_paged_attention_workspace_bytes"], ctypes.c_int64
    return f


@pytest.mark.parametrize("T,R,H,HK,D,max_q", [
    (8192, 4, 32, 8, 128, 0), (8192, 1, 32, 8, 128, 0), (8192, 4, 32, 8, 64, 0),
    (32768, 20, 32, 8, 128, 0), (60000, 100, 32, 8, 128, 0), (66000, 4, 64, 32, 128, 0),
    (32768, 4, 64, 64, 128, 0), (1000, 1000, 32, 8, 128, 1), (4096, 4096, 32, 8, 128, 1),
    (4096, 4096, 32, 32, 64, 1), (2500, 2500, 32, 32, 128, 1),
])
def test_scratch_of_uncut_blocks(query, T, R, H, HK, D, max_q):
    """Prompts that fill the chip are not cut, nor are most of many decoding
    requests. At most one and a half rounds of the chip's 512 to 1024 workgroups are
    chunks of cut blocks, and as many the short ones at their ends: a state each of 32
    columns of D sums and two statistics (in 128 words). The list of the work past 192
    requests comes on top, 40 bytes an item."""
    state = (32 * D + 128) * 4
    chunks = 2 * 1.5 * 256 * (2 if D == 128 else 4)
    got = query(T, R, 512, H, HK, D, 64, max_q)
    # a long decoding request beside them can still be cut
    assert got > hip.PAGED_ZERO_BYTES + 2 * HK * state
    assert got <= hip.PAGED_ZERO_BYTES + chunks * state + 40 * 65536


def test_scratch_of_cut_prompts(query):
    """A mixed step of 36 requests, and 512 tokens behind 15872 keys."""
    assert 10 * MB < query(512, 1, 256, 32, 8, 128, 64, 0) <= 100 * MB
    assert query(1800, 36, 64, 32, 8, 128, 64, 512) <= 100 * MB


def test_no_scratch_where_nothing_is_cut(query):
    assert query(1, 1, 2, 32, 8, 128, 64, 1) == 0      # a table of 128 keys
    assert query(64, 64, 8, 32, 8, 128, 16, 1) == 0
