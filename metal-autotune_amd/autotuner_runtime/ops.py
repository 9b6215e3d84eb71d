"""Tensor-level ops on the gfx950 library: the library calls the reference's
regions splice around (mx.quantized_matmul, mx.dequantize, mx.fast.rms_norm,
mx.fast.rope, mx.fast.scaled_dot_product_attention, mlx-lm's swiglu and
quantized embedding, LFM2's short-conv) plus the fused region entry points.

Every function allocates its outputs with torch on the inputs' device and
launches on torch's current stream; none synchronizes. They run only on GPU
tensors (hip.lib() raises otherwise); there is no CPU path.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from typing import NamedTuple

import torch

from . import hip


def _empty(shape, like: torch.Tensor, dtype=None) -> torch.Tensor:
    return like.new_empty(shape, dtype=dtype)


def _qp(group_size: int, bits: int) -> dict:
    return {"group_size": group_size, "bits": bits}


# -- A1 ---------------------------------------------------------------------

def dequantize(w, scales, biases, group_size: int = 64, bits: int = 4) -> torch.Tensor:
    """mx.dequantize (affine): T(fma(s, q, b)) as [N, K] in the scales' dtype."""
    N, K = w.shape[0], w.shape[1] * 32 // bits
    out = _empty((N, K), scales)
    hip.b_dequant([w, scales, biases], [out], _qp(group_size, bits))
    return out


def quantized_embedding(ids, w, scales, biases, group_size: int = 64, bits: int = 4):
    """nn.QuantizedEmbedding: dequantized rows ids -> [*ids.shape, K]."""
    K = w.shape[1] * 32 // bits
    out = _empty((*ids.shape, K), scales)
    hip.b_gather_dequant([ids.contiguous(), w, scales, biases], [out], _qp(group_size, bits))
    return out


# -- A2-A4 and the qmm regions ---------------------------------------------

def quantized_matmul(x, w, scales, biases, transpose: bool = True, group_size: int = 64,
                     bits: int = 4, mode: str = "affine") -> torch.Tensor:
    """mx.quantized_matmul(x, w, scales, biases, transpose=True, group_size, bits,
    mode='affine') -> x @ dequant(w)^T."""
    if not transpose or mode != "affine":
        raise ValueError("only transpose=True, mode='affine' is covered (the MLX checkpoint layout)")
    y = _empty((*x.shape[:-1], w.shape[0]), x)
    hip.b_qmm([x.contiguous(), w, scales, biases], [y], _qp(group_size, bits))
    return y


def qmm_residual(x, w, scales, biases, resid, group_size=64, bits=4):
    """Region [qmm, add]: T(resid + T(x @ W^T))."""
    y = _empty((*x.shape[:-1], w.shape[0]), x)
    hip.b_qmm_residual([x.contiguous(), w, scales, biases, resid.contiguous()], [y],
                       _qp(group_size, bits))
    return y


def qmm_residual_rmsnorm(x, w, scales, biases, resid, norm_w, eps: float, group_size=64, bits=4):
    """Region [qmm, add, rms_norm] -> (h, rms_norm(h))."""
    shape = (*x.shape[:-1], w.shape[0])
    h, y = _empty(shape, x), _empty(shape, x)
    hip.b_qmm_residual_rmsnorm([x.contiguous(), w, scales, biases, resid.contiguous(), norm_w],
                               [h, y], {**_qp(group_size, bits), "eps": eps})
    return h, y


def qmm_split_gate(x, w, scales, biases, group_size=64, bits=4):
    """Region [qmm, split(3), mul] -> (C, T(B * x))."""
    shape = (*x.shape[:-1], w.shape[0] // 3)
    c, bx = _empty(shape, x), _empty(shape, x)
    hip.b_qmm_split_gate([x.contiguous(), w, scales, biases], [c, bx], _qp(group_size, bits))
    return c, bx


def qmm_dual(x, w1, s1, b1, w2, s2, b2, group_size=64, bits=4, swiglu: bool = False):
    """Region [qmm(w1), qmm(w3)] -> (x W1^T, x W3^T), or swiglu of the two."""
    shape = (*x.shape[:-1], w1.shape[0])
    p = {**_qp(group_size, bits), "act": hip.MI_ACT_SWIGLU if swiglu else hip.MI_ACT_NONE}
    ins = [x.contiguous(), w1, s1, b1, w2, s2, b2]
    if swiglu:
        y = _empty(shape, x)
        hip.b_qmm_dual(ins, [y], p)
        return y
    y1, y2 = _empty(shape, x), _empty(shape, x)
    hip.b_qmm_dual(ins, [y1, y2], p)
    return y1, y2


def qmm_grouped3(x, weights, group_size=64, bits=4):
    """Three projections of one x in one launch: ``weights`` is three
    (w, scales, biases) triples; returns the three x @ dequant(w)^T."""
    outs = [_empty((*x.shape[:-1], w.shape[0]), x) for w, _, _ in weights]
    ins = [x.contiguous()] + [t for triple in weights for t in triple]
    hip.b_qmm_grouped3(ins, outs, _qp(group_size, bits))
    return outs


# -- A5, A6 ----------------------------------------------------------------

def rms_norm(x, weight, eps: float) -> torch.Tensor:
    """mx.fast.rms_norm over the last axis."""
    x = x.contiguous()
    y = torch.empty_like(x)
    hip.b_rms_norm([x, weight], [y], {"eps": eps})
    return y


def norm_rope(x, weight, n_heads: int, eps: float, dims: int, base: float, offset: int = 0,
              traditional: bool = False, scale: float = 1.0, out: torch.Tensor | None = None,
              out_pos: int = 0) -> torch.Tensor:
    """reshape(B, L, H, D) -> rms_norm(weight) (skipped if None) -> transpose(0,2,1,3)
    -> mx.fast.rope(dims, traditional, base, scale, offset). With ``out`` (a
    [B, H, cap, D] cache) the rows land at [out_pos, out_pos + L) in place."""
    x = x.contiguous()
    B, L, HD = x.shape
    D = HD // n_heads
    if out is None:
        out = _empty((B, n_heads, L, D), x)
        cap, pos = L, 0
    else:
        if not out.is_contiguous() or out.shape[0] != B or out.shape[1] != n_heads or out.shape[3] != D:
            raise ValueError(f"cache target {tuple(out.shape)} does not hold {(B, n_heads, '*', D)}")
        cap, pos = out.shape[2], out_pos
    if weight is not None and (tuple(weight.shape) != (D,) or weight.dtype != x.dtype):
        raise ValueError(f"norm weight must be {x.dtype} [{D}]")
    hip._require_gpu(x)
    hip._check(hip.lib().mi_norm_rope(
        x.data_ptr(), None if weight is None else weight.data_ptr(), out.data_ptr(), B, L,
        n_heads, D, HD, float(eps), int(dims), int(traditional), float(base), float(scale),
        int(offset), cap, pos, hip._dt(x), hip._stream(x)), "norm_rope")
    return out


def norm_rope_qkv(q, k, v, q_norm, k_norm, n_heads: int, n_kv_heads: int, eps: float, dims: int,
                  base: float, offset: int, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  cache_pos: int, traditional: bool = False, scale: float = 1.0) -> torch.Tensor:
    """The attention prologue in one launch: q -> rms_norm -> rope -> [B, H, L, D]
    (returned); k -> rms_norm -> rope and v -> transpose, written into the
    caches at rows [cache_pos, cache_pos + L). Equal bit for bit to three
    norm_rope calls. q, k, v may be row-strided views ([B, L, H*D] slices)."""
    B, L, _ = q.shape
    D = q.shape[-1] // n_heads
    for t, h in ((k, n_kv_heads), (v, n_kv_heads)):
        if t.shape[:2] != (B, L) or t.shape[-1] != h * D or t.dtype != q.dtype:
            raise ValueError("q, k and v must share batch, length, head dim and dtype")
    for t in (q, k, v):
        if t.stride(-1) != 1 or t.stride(0) != L * t.stride(1):
            raise ValueError("q, k, v rows must be unit-stride with a uniform row stride")
    for c in (k_cache, v_cache):
        if (not c.is_contiguous() or c.shape[0] != B or c.shape[1] != n_kv_heads
                or c.shape[3] != D or c.dtype != q.dtype):
            raise ValueError(f"cache {tuple(c.shape)} does not hold {(B, n_kv_heads, '*', D)}")
    for wt in (q_norm, k_norm):
        if tuple(wt.shape) != (D,) or wt.dtype != q.dtype:
            raise ValueError(f"norm weight must be {q.dtype} [{D}]")
    out = _empty((B, n_heads, L, D), q)
    hip._require_gpu(q)
    hip._check(hip.lib().mi_norm_rope_qkv(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(1), k.stride(1), v.stride(1),
        q_norm.data_ptr(), k_norm.data_ptr(), out.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), B, L, n_heads, n_kv_heads, D, float(eps), int(dims),
        int(traditional), float(base), float(scale), int(offset), k_cache.shape[2],
        int(cache_pos), hip._dt(q), hip._stream(q)), "norm_rope_qkv")
    return out


def qkv_norm_rope(x, weights, q_norm, k_norm, n_heads: int, n_kv_heads: int, eps: float,
                  dims: int, base: float, offset: int, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, cache_pos: int, group_size: int = 64, bits: int = 4,
                  traditional: bool = False, scale: float = 1.0) -> torch.Tensor | None:
    """The q/k/v projections and the attention prologue in one launch:
    ``norm_rope_qkv(*qmm_grouped3(x, weights), ...)`` bit for bit, without
    writing q, k and v (patch/wrappers.py:156-176). ``weights`` is the (w,
    scales, biases) triples of q, k and v. Returns q_out [B, Hq, L, D] (k and v
    go into the caches at rows [cache_pos, cache_pos + L)), or None when the
    fused entry does not cover these shapes -- the caller then runs the two
    ops."""
    if x.dim() != 3:
        raise ValueError(f"x must be [B, L, K], got {tuple(x.shape)}")
    B, L, _ = x.shape
    p = _qp(group_size, bits)
    Ns = [hip._qmm_dims(x, w, s, b, p)[1] for w, s, b in weights]
    if Ns[0] % n_heads or Ns[1] % n_kv_heads or Ns[2] != Ns[1]:
        raise ValueError(f"projection widths {Ns} do not split into {n_heads} / {n_kv_heads} heads")
    D = Ns[0] // n_heads
    if Ns[1] // n_kv_heads != D:
        raise ValueError("q and k/v heads must share a head dim")
    for c in (k_cache, v_cache):
        if (not c.is_contiguous() or c.dim() != 4 or c.shape[0] != B
                or c.shape[1] != n_kv_heads or c.shape[3] != D or c.dtype != x.dtype):
            raise ValueError(f"cache {tuple(c.shape)} does not hold {(B, n_kv_heads, '*', D)}")
    for wt in (q_norm, k_norm):
        if tuple(wt.shape) != (D,) or wt.dtype != x.dtype or not wt.is_contiguous():
            raise ValueError(f"norm weight must be contiguous {x.dtype} [{D}]")
    hip._require_gpu(x)
    x = x.contiguous()
    hip._contig(*[t for triple in weights for t in triple])
    dt = hip._act_dtype(x, weights[0][1])
    out = _empty((B, n_heads, L, D), x)
    ptrs = ctypes.c_void_p * 3
    status = hip.lib().mi_qmm_affine_qkv_norm_rope(
        x.data_ptr(), ptrs(*[w.data_ptr() for w, _, _ in weights]),
        ptrs(*[s.data_ptr() for _, s, _ in weights]), ptrs(*[b.data_ptr() for _, _, b in weights]),
        q_norm.data_ptr(), k_norm.data_ptr(), out.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), B, L, n_heads, n_kv_heads, D, x.shape[-1], group_size, bits,
        float(eps), int(dims), int(traditional), float(base), float(scale), int(offset),
        k_cache.shape[2], int(cache_pos), dt, hip._stream(x))
    if status == hip.MI_ERR_UNSUPPORTED:
        return None
    hip._check(status, "qkv_norm_rope")
    return out


def rope(x, dims: int, traditional: bool = False, base: float = 10000.0, scale: float = 1.0,
         offset: int = 0) -> torch.Tensor:
    """mx.fast.rope on [..., L, D] (the position axis is -2)."""
    x = x.contiguous()
    L, D = x.shape[-2], x.shape[-1]
    lead = x.numel() // (L * D) if L * D else 0
    flat = x.reshape(lead, L, D)  # one "head" per leading index: [B', L, 1*D]
    out = norm_rope(flat, None, 1, 0.0, dims, base, offset, traditional, scale)
    return out.reshape(x.shape)


def write_kv(v, n_heads: int, cache: torch.Tensor, pos: int) -> None:
    """The value half of a KV cache's update_and_fetch: reshape(B, L, H, D),
    transpose(0, 2, 1, 3), written into cache rows [pos, pos + L)."""
    norm_rope(v, None, n_heads, 0.0, 0, 1.0, 0, out=cache, out_pos=pos)


# -- A7 --------------------------------------------------------------------

def scaled_dot_product_attention(q, k, v, scale: float, mask: str | None = "causal",
                                 kv_len: int | None = None, out_layout: int = 0):
    """mx.fast.scaled_dot_product_attention(q, k, v, scale, mask='causal'|None).
    q [B, H, Lq, D]; k, v [B, HK, cap, D] with the first ``kv_len`` rows valid
    (default: all). out_layout 1 returns [B, Lq, H, D] (the transpose before
    o_proj, fused)."""
    if mask not in ("causal", None):
        raise ValueError("mask must be 'causal' or None")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    B, H, Lq, D = q.shape
    HK, cap = k.shape[1], k.shape[2]
    Lk = cap if kv_len is None else int(kv_len)
    o = _empty((B, H, Lq, D) if out_layout == 0 else (B, Lq, H, D), q)
    hip._require_gpu(q)
    if tuple(v.shape) != tuple(k.shape) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("k and v must match each other and q's dtype")
    hip.sdpa(q, k, v, o, Lk, cap, float(scale), int(mask == "causal"), int(out_layout))
    return o


# -- A8-A10, A12 -------------------------------------------------------------

def swiglu(g, u) -> torch.Tensor:
    """mlx_lm.models.activations.swiglu(gate, up) = silu(gate) * up."""
    g, u = g.contiguous(), u.contiguous()
    y = torch.empty_like(g)
    hip.b_swiglu([g, u], [y], {})
    return y


def shortconv(bx, c, w, state=None):
    """LFM2 short-conv core -> (T(c * conv(concat(state, bx))), new state [B, 2, D])."""
    bx, c = bx.contiguous(), c.contiguous()
    out = torch.empty_like(bx)
    st = _empty((bx.shape[0], 2, bx.shape[2]), bx)
    ins = [bx, c, w.contiguous()] + ([state.contiguous()] if state is not None else [])
    hip.b_shortconv(ins, [out, st], {})
    return out, st


def linear_f32(x, w, bias=None, gelu: bool = False) -> torch.Tensor:
    """nn.Linear in fp32 (mx.addmm(b, x, W^T)), optionally followed by exact GELU."""
    x = x.contiguous()
    y = _empty((*x.shape[:-1], w.shape[0]), x)
    ins = [x, w.contiguous()] + ([bias.contiguous()] if bias is not None else [])
    hip.b_linear_f32(ins, [y], {"act": hip.MI_ACT_GELU if gelu else hip.MI_ACT_NONE})
    return y


def gelu_mlp_f32(x, w1, b1, w2, b2) -> torch.Tensor:
    """Config 1's tiny MLP in one launch: gelu(x W1^T + b1) W2^T + b2 (fp32)."""
    x = x.contiguous()
    y = _empty((x.shape[0], w2.shape[0]), x)
    hip.b_gelu_mlp_f32([x, w1.contiguous(), b1.contiguous(), w2.contiguous(), b2.contiguous()],
                       [y], {})
    return y


def argmax(x, split: bool = True) -> torch.Tensor:
    """Greedy token: argmax over the last axis (lowest index on ties) as int32.
    split: each row over many workgroups (default) or one workgroup per row;
    the result is the same."""
    x = x.contiguous()
    o = _empty(x.shape[:-1], x, torch.int32)
    hip.b_argmax([x], [o], {"split": split})
    return o


# -- several requests over a paged KV cache (no counterpart in the reference) ----
#
# Pools of pages k_pages, v_pages [n_pages, HK, page_size, D]; a block table int32
# [R, width] of each request's pages; the tokens of a step request after request.

_I32, _F32 = torch.int32, torch.float32


def _i32(what: str, dev: int, *arrays) -> None:
    for t in arrays:
        if t.dtype is not _I32 or t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"{what}: lengths, tables and positions must be contiguous int32 "
                             f"arrays on one device, got {t.dtype} {tuple(t.shape)} on {t.device}")


_HERE = contextlib.nullcontext()


def _on(dev: int):
    """The tensors' device as the current one, for the launch."""
    return _HERE if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)


class PagedPlan(NamedTuple):
    """One step's bookkeeping, on the GPU (``paged_plan``)."""

    cu_q: torch.Tensor        # int32 [R + 1]: where each request's tokens start
    kv_lens: torch.Tensor     # int32 [R]: its keys after the step, 0 if refused
    positions: torch.Tensor   # int32 [num_tokens]: each token's position in its request
    slots: torch.Tensor       # int32 [num_tokens]: its cache slot, -1 if it has none
    free_count: torch.Tensor  # int32 [1]: the free pages that remain
    refused: torch.Tensor     # int32 [1]: requests that got no pages


def paged_plan(block_table, kv_lens, q_lens, free_pages, free_count, page_size: int,
               num_tokens: int, out: PagedPlan | None = None) -> PagedPlan:
    """A step's bookkeeping in one launch: request r holds kv_lens[r] keys and
    brings q_lens[r] tokens (int32 [R]); the pages it lacks are taken from the end
    of free_pages[:free_count] (int32 [F], int32 [1]), request after request, and
    written into block_table (int32 [R, width]) in place. num_tokens: rows of the
    step's token buffer (rows behind the sum of q_lens get position 0 and slot -1).
    A request whose pages are not there, whose keys would pass its row of the table
    or whose tokens those rows, takes none and is counted in ``refused``. out: an earlier
    plan of as many requests and tokens, written again (a captured graph reads it
    where it is); its kv_lens and free_count may not be this call's inputs."""
    shape = kv_lens.shape
    if block_table.dim() != 2 or len(shape) != 1 or q_lens.shape != shape \
            or shape[0] != block_table.shape[0] or free_pages.dim() != 1 \
            or free_count.numel() != 1:
        raise ValueError("paged_plan takes block_table [R, width], kv_lens [R], q_lens [R], "
                         "free_pages [F] and free_count [1]")
    dev = block_table.get_device()
    _i32("paged_plan", dev, block_table, kv_lens, q_lens, free_pages, free_count)
    R, width = block_table.shape
    T = int(num_tokens)
    if T < 0:
        raise ValueError(f"paged_plan: num_tokens={T}")
    if not block_table.is_cuda:
        hip._require_gpu(block_table)
    if out is None:
        # one allocation for the six outputs, which lie one after another
        buf = block_table.new_empty(2 * (R + T) + 3)
        at = buf.data_ptr()
        ptrs = (at, at + 4 * (R + 1), at + 4 * (2 * R + 1), at + 4 * (2 * R + 1 + T),
                at + 4 * (2 * (R + T) + 1), at + 4 * (2 * (R + T) + 2))
        out = PagedPlan._make(torch.split_with_sizes(buf, (R + 1, R, T, T, 1, 1)))
    else:
        if [t.numel() for t in out] != [R + 1, R, T, T, 1, 1]:
            raise ValueError(f"paged_plan: out is not a plan of {R} requests and {T} tokens")
        _i32("paged_plan", dev, *out)
        ptrs = [t.data_ptr() for t in out]
        if ptrs[1] == kv_lens.data_ptr() or ptrs[4] == free_count.data_ptr():
            raise ValueError("paged_plan: out holds this call's inputs")
    with _on(dev):
        hip._check(hip.lib().mi_paged_plan(
            block_table.data_ptr(), width, kv_lens.data_ptr(), q_lens.data_ptr(),
            free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), R, T,
            int(page_size), *ptrs, hip._stream(block_table)), "paged_plan")
    return out


def rope_table(dims: int, base: float = 10000.0, scale: float = 1.0, freqs=None,
               device="cuda") -> torch.Tensor:
    """The angle per position of each rotation pair, fp64 [dims / 2], made once and
    kept: scale * base^(-2 i / dims), or scale / freqs[i] where ``freqs`` is given
    (mx.fast.rope's argument: long-context scalings that stretch each wavelength
    differently)."""
    if freqs is not None:
        f = torch.as_tensor(freqs, dtype=torch.float64, device=device)
        if tuple(f.shape) != (dims // 2,):
            raise ValueError(f"freqs must hold {dims // 2} values, got {tuple(f.shape)}")
        return scale / f
    i = torch.arange(dims // 2, dtype=torch.float64, device=device)
    return scale * base ** (-2.0 * i / dims)


def _paged_pools(what: str, q, k_pages, v_pages, D: int):
    shape, dt, dev = k_pages.shape, q.dtype, q.get_device()
    if len(shape) != 4 or v_pages.shape != shape or shape[3] != D or k_pages.dtype is not dt \
            or v_pages.dtype is not dt or k_pages.get_device() != dev \
            or v_pages.get_device() != dev or not k_pages.is_contiguous() \
            or not v_pages.is_contiguous():
        raise ValueError(f"{what}: the pools must be contiguous {dt} [pages, heads, page size, "
                         f"{D}] on {q.device}, got {tuple(shape)} and {tuple(v_pages.shape)}")
    return shape


def norm_rope_paged(q, k, v, q_norm, k_norm, n_heads: int, n_kv_heads: int, eps: float,
                    inv_freq, positions, slots, k_pages, v_pages,
                    traditional: bool = False) -> torch.Tensor:
    """The attention prologue of a step's tokens in one launch: q [T, H * D] ->
    rms_norm(q_norm) -> rope -> [T, H, D] (returned); k -> rms_norm(k_norm) -> rope
    and v, written to each token's slot of the pools (none where the slot is -1).
    A norm weight of None skips the normalization. ``inv_freq``: ``rope_table``'s,
    whose 2 * len(inv_freq) leading values of a head are turned, at the angle of
    each token's own position. q, k, v may be column ranges of one projection."""
    T, width = q.shape
    D = width // n_heads
    dt, dev, kv = q.dtype, q.get_device(), (T, n_kv_heads * D)
    if width != n_heads * D or k.shape != kv or v.shape != kv or k.dtype is not dt \
            or v.dtype is not dt or k.get_device() != dev or v.get_device() != dev:
        raise ValueError(f"norm_rope_paged: q, k, v must be one type on one device, [T, heads * D], "
                         f"got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    for wt in (q_norm, k_norm):
        if wt is not None and (wt.shape != (D,) or wt.dtype is not dt or wt.get_device() != dev
                               or not wt.is_contiguous()):
            raise ValueError(f"norm weight must be contiguous {dt} [{D}] on {q.device}")
    n_pages, hk, page, _ = _paged_pools("norm_rope_paged", q, k_pages, v_pages, D)
    if hk != n_kv_heads or positions.shape != (T,) or slots.shape != (T,):
        raise ValueError(f"norm_rope_paged: pools of {n_kv_heads} heads, positions and slots of "
                         f"{T} tokens are needed")
    _i32("norm_rope_paged", dev, positions, slots)
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 \
            or inv_freq.get_device() != dev or not inv_freq.is_contiguous():
        raise ValueError("norm_rope_paged: inv_freq must be a float64 array (ops.rope_table)")
    if not q.is_cuda:
        hip._require_gpu(q)
    (sq, uq), (sk, uk), (sv, uv) = q.stride(), k.stride(), v.stride()
    pq, pk, pv = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (pq | pk | pv) & 15 or (sq | sk | sv) & 7 or not uq == uk == uv == 1:
        # rows the kernel cannot read in 16-byte pieces are copied first
        q, k, v = (t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
        (sq, _), (sk, _), (sv, _) = q.stride(), k.stride(), v.stride()
        pq, pk, pv = q.data_ptr(), k.data_ptr(), v.data_ptr()
    out = q.new_empty((T, n_heads, D))
    with _on(dev):
        hip._check(hip.lib().mi_norm_rope_paged(
            pq, pk, pv, sq, sk, sv, None if q_norm is None else q_norm.data_ptr(),
            None if k_norm is None else k_norm.data_ptr(), out.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), inv_freq.data_ptr(), 2 * inv_freq.shape[0], int(traditional),
            positions.data_ptr(), slots.data_ptr(), T, n_heads, n_kv_heads, D, n_pages, page,
            eps, hip._dt(q), hip._stream(q)), "norm_rope_paged")
    return out


def paged_attention(q, k_pages, v_pages, block_table, cu_q, kv_lens, scale: float,
                    max_q_len: int | None = None) -> torch.Tensor:
    """Causal GQA attention of every request's new tokens over its pages, one call
    for requests of any lengths: q [T, H, D] -> [T, H, D]. Request r's tokens are
    rows [cu_q[r], cu_q[r + 1]), its keys kv_lens[r], these tokens' own among them
    (``paged_plan``'s cu_q and kv_lens). max_q_len: the most tokens a request
    brings, where the caller knows it: it chooses the kernels, never the result's
    meaning. Rows behind the last request's are not written."""
    if q.dim() != 3:
        raise ValueError(f"paged_attention: q must be [T, H, D], got {tuple(q.shape)}")
    _paged_pools("paged_attention", q, k_pages, v_pages, q.shape[2])
    R, = kv_lens.shape
    if block_table.dim() != 2 or block_table.shape[0] != R or cu_q.shape != (R + 1,):
        raise ValueError("paged_attention takes block_table [R, width], cu_q [R + 1], kv_lens [R]")
    dev = q.get_device()
    _i32("paged_attention", dev, block_table, cu_q, kv_lens)
    if not q.is_cuda:
        hip._require_gpu(q)
    if not q.is_contiguous() or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_like(q)
    with _on(dev):
        hip.paged_attention(q, k_pages, v_pages, out, block_table, cu_q, kv_lens, scale,
                            0 if max_q_len is None else max_q_len)
    return out


class TokenLogprobs(NamedTuple):
    """``token_logprobs``' results, fp32 (ids int32)."""

    logprobs: torch.Tensor      # [rows]
    entropy: torch.Tensor       # [rows]
    top_ids: torch.Tensor       # [rows, top]
    top_logprobs: torch.Tensor  # [rows, top]


def token_logprobs(logits, tokens, top: int = 0) -> TokenLogprobs:
    """Log probabilities of given tokens: logits [..., V], tokens [...] -> each
    row's log softmax at its token (NaN outside [0, V)), its entropy, and its
    ``top`` (0 to 64) most probable tokens with their log probabilities, the lowest
    index first among equal logits. Logits of -inf are forbidden tokens."""
    if not logits.is_cuda:
        hip._require_gpu(logits)
    shape = logits.shape
    lead, V = shape[:-1], shape[-1]
    wide = tokens.dtype is torch.int64
    if tokens.shape != lead or not (wide or tokens.dtype is _I32) \
            or tokens.get_device() != logits.get_device():
        raise ValueError(f"token_logprobs: tokens must be int32 or int64 {tuple(lead)} on "
                         f"{logits.device}")
    if not 0 <= top <= 64 or top > V or V < 1:
        raise ValueError(f"token_logprobs: top={top} of V={V} (0 to 64, at most V)")
    x = logits
    if not x.is_contiguous() and (x.stride(-1) != 1 or len(lead) != 1):
        x = x.contiguous()
    if len(lead) != 1:
        x = x.reshape(-1, V)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    logprobs = x.new_empty(lead, dtype=_F32)
    out = TokenLogprobs(logprobs, torch.empty_like(logprobs),
                        x.new_empty((*lead, top), dtype=_I32),
                        logprobs.new_empty((*lead, top)))
    with _on(x.get_device()):
        hip.token_logprobs(x, tokens, wide, top, *out)
    return out


# -- several continuations of a prompt (no counterpart in the reference) ----------

class BeamStep(NamedTuple):
    """``beam_select``'s choice, [R, width] each, the best first."""

    scores: torch.Tensor    # fp32; -inf where there were fewer candidates
    parents: torch.Tensor   # int32: the row of the logits that each continues
    tokens: torch.Tensor    # int32: the token that it continues with
    finished: torch.Tensor  # bool


def beam_select(logits, scores, width: int | None = None, finished=None,
                eos: int | None = None) -> BeamStep:
    """Beam search's choice: of R prompts of B beams each the ``width`` (default B, 1 to
    64) best continuations over beams and vocabulary. logits [R * B, V], beam after beam
    of prompt after prompt; scores fp32 [R, B], to which the candidates' log probabilities
    are added (-inf: a beam that offers nothing, as all but one are at the first step).
    finished [R, B] (bool): beams that have ended offer themselves alone, with the token
    ``eos`` at their own score. The best first; among equal ones the lowest beam, then the
    lowest token. Candidates of different beams are compared in 64 bits. Where there are
    fewer than ``width``, the rest has score -inf, the prompt's first beam and token 0."""
    if not logits.is_cuda:
        hip._require_gpu(logits)
    dev = logits.get_device()
    if scores.dim() != 2 or scores.dtype is not _F32 or scores.get_device() != dev \
            or not scores.is_contiguous():
        raise ValueError(f"beam_select: scores must be a contiguous float32 [prompts, beams] on "
                         f"{logits.device}, got {scores.dtype} {tuple(scores.shape)}")
    R, B = scores.shape
    if logits.dim() != 2 or logits.shape[0] != R * B:
        raise ValueError(f"beam_select: logits must be [{R * B}, V], got {tuple(logits.shape)}")
    if finished is not None:
        if finished.shape != scores.shape or finished.dtype is not torch.bool \
                or finished.get_device() != dev or not finished.is_contiguous():
            raise ValueError(f"beam_select: finished must be a contiguous bool {(R, B)} on "
                             f"{logits.device}")
        if eos is None:
            raise ValueError("beam_select: finished beams need the token eos")
    K = B if width is None else int(width)
    if K < 1:
        raise ValueError(f"beam_select: width={K}")
    x = logits if logits.stride(1) == 1 and logits.stride(0) >= 0 else logits.contiguous()
    parents = x.new_empty((R, K), dtype=_I32)
    out = BeamStep(scores.new_empty((R, K)), parents, torch.empty_like(parents),
                   x.new_empty((R, K), dtype=torch.bool))
    with _on(dev):
        hip.beam_select(x, scores, finished, -1 if eos is None else eos, K, *out)
    return out


FORK_MAX_PAGES = 1 << 20  # that paged_fork and paged_compact cover


class PagePools(NamedTuple):
    """The pools of all layers as ``paged_fork`` and ``paged_compact`` take them
    (``page_pools``)."""

    pointers: torch.Tensor  # int64, on the device: where each begins
    pools: tuple            # the pools, kept alive
    shape: tuple            # (pages, heads, page size, bytes of a row)


def page_pools(pools) -> PagePools:
    """Pools [pages, heads, page size, head dim] of one shape and type on one device
    (every layer's k_pages and v_pages), made once and kept: whatever pages a fork or a
    compaction moves, it moves in all of them. Both cover pools of FORK_MAX_PAGES pages."""
    pools = tuple(pools)
    if not pools:
        raise ValueError("page_pools: no pools")
    first = pools[0]
    if not first.is_cuda:
        hip._require_gpu(first)
    for p in pools:
        if p.dim() != 4 or p.shape != first.shape or p.dtype is not first.dtype \
                or p.get_device() != first.get_device() or not p.is_contiguous() \
                or p.data_ptr() & 15:
            raise ValueError(f"page_pools: the pools must be contiguous, 16-byte aligned "
                             f"{first.dtype} {tuple(first.shape)} on {first.device}, got {p.dtype} "
                             f"{tuple(p.shape)} on {p.device}")
    n, heads, page, D = first.shape
    pointers = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64).to(first.device)
    return PagePools(pointers, pools, (n, heads, page, D * first.element_size()))


def _check_pages(what: str, pools: PagePools, block_table, kv_lens, free_pages, free_count,
                 *more) -> int:
    dev = pools.pointers.get_device()
    if block_table.dim() != 2 or kv_lens.shape != block_table.shape[:1] or free_pages.dim() != 1 \
            or free_count.numel() != 1 or any(t.shape != kv_lens.shape for t in more):
        raise ValueError(f"{what} takes block_table [R, width], an entry of [R] a request, "
                         "free_pages [F] and free_count [1]")
    _i32(what, dev, block_table, kv_lens, free_pages, free_count, *more)
    if not block_table.shape[0]:
        raise ValueError(f"{what}: no requests")
    return dev


def paged_fork(block_table, kv_lens, sources, free_pages, free_count,
               pools: PagePools) -> torch.Tensor:
    """Requests that go on from others' keys: request r continues request sources[r]
    (int32 [R]; itself, too), or ends where that is negative. Full pages are shared from
    then on, a part-filled last one stays with one of those that go on from it and is
    copied for the others, in every layer's pools; pages that nobody holds any more go
    back to the free list first (in the order of their ids), and the copies' pages come
    from its end. block_table, kv_lens, free_pages (of as many entries as there are pages)
    and free_count are changed in place. Returns int32 [1]: 0, or how many pages were
    missing (sources past the last request count as such); then nothing has changed.
    Shared pages are full: the next step's tokens never fall into them."""
    dev = _check_pages("paged_fork", pools, block_table, kv_lens, free_pages, free_count, sources)
    refused = kv_lens.new_empty(1)
    with _on(dev):
        hip.paged_fork(block_table, kv_lens, sources, free_pages, free_count, refused, pools)
    return refused


def paged_compact(block_table, kv_lens, free_pages, free_count, pools: PagePools) -> torch.Tensor:
    """The pages that requests hold moved to the lowest ids, in every layer's pools:
    block_table, free_pages (of as many entries as there are pages) and free_count are
    changed in place; every page that no request holds is free afterwards, the highest
    first in the list. Returns int32 [1]: how many are held. To a step one free page is as
    good as another; this is for caches that are to be stored or moved, which are then the
    first pages of each pool, or cut: requests go on in copies of the pools' first P pages
    of N with free_pages[N - P:] and free_count - (N - P)."""
    dev = _check_pages("paged_compact", pools, block_table, kv_lens, free_pages, free_count)
    live = kv_lens.new_empty(1)
    with _on(dev):
        hip.paged_compact(block_table, kv_lens, free_pages, free_count, live, pools)
    return live


class SharedPlan(NamedTuple):
    """A step's plan of attention behind shared prefixes (``paged_shared_plan``)."""

    keys: torch.Tensor      # int32 [groups]: the leading keys that all of a group hold alike
    schedule: torch.Tensor  # the work, for ``paged_shared_attention``
    shape: tuple            # (T, R, groups, width, H, HK, D, page size): what it is for


def paged_shared_plan(block_table, cu_q, kv_lens, cu_groups, page_size: int, num_tokens: int,
                      n_heads: int, n_kv_heads: int, head_dim: int,
                      out: SharedPlan | None = None) -> SharedPlan:
    """What groups of requests share, and a step's attention laid out for it, once for all
    layers: group g is the requests [cu_groups[g], cu_groups[g + 1]) (int32 [groups + 1];
    requests outside all groups are by themselves), whose common leading keys are found
    from block_table's rows: whole pages, cached before the step, that all of the group's
    requests hold. block_table, cu_q, kv_lens: a step's, as ``paged_attention`` takes them
    (``paged_plan`` makes them), of num_tokens rows. out: an earlier plan of these sizes,
    written again (a captured graph reads it where it is)."""
    R, = kv_lens.shape
    if block_table.dim() != 2 or block_table.shape[0] != R or cu_q.shape != (R + 1,) \
            or cu_groups.dim() != 1 or cu_groups.shape[0] < 2:
        raise ValueError("paged_shared_plan takes block_table [R, width], cu_q [R + 1], kv_lens [R] "
                         "and cu_groups [groups + 1]")
    dev = block_table.get_device()
    _i32("paged_shared_plan", dev, block_table, cu_q, kv_lens, cu_groups)
    if not block_table.is_cuda:
        hip._require_gpu(block_table)
    shape = (int(num_tokens), R, cu_groups.shape[0] - 1, block_table.shape[1], int(n_heads),
             int(n_kv_heads), int(head_dim), int(page_size))
    if out is None:
        n = hip.shared_plan_ints(*shape)
        buf = block_table.new_empty(n + shape[2])
        out = SharedPlan(buf[n:], buf[:n], shape)
    elif out.shape != shape or out.schedule.get_device() != dev:
        raise ValueError(f"paged_shared_plan: out is a plan for {out.shape}, not {shape}")
    with _on(dev):
        hip.paged_shared_plan(block_table, cu_q, kv_lens, cu_groups, out)
    return out


def paged_shared_attention(q, k_pages, v_pages, block_table, plan: SharedPlan,
                           scale: float) -> torch.Tensor:
    """``paged_attention`` of the step that ``plan`` was made for, with the keys that a
    group's requests share read once for all of them: q [T, H, D] -> [T, H, D]. The same
    results within rounding. block_table: the plan's. Rows behind the last request's are
    not written."""
    T, R, _, width, H, HK, D, page = plan.shape
    if q.shape != (T, H, D):
        raise ValueError(f"paged_shared_attention: the plan is for q {(T, H, D)}, got "
                         f"{tuple(q.shape)}")
    _, hk, rows, _ = _paged_pools("paged_shared_attention", q, k_pages, v_pages, D)
    if hk != HK or rows != page or block_table.shape != (R, width):
        raise ValueError(f"paged_shared_attention: the plan is for pages of {HK} heads of {page} rows "
                         f"and a table {(R, width)}")
    dev = q.get_device()
    _i32("paged_shared_attention", dev, block_table, plan.schedule)
    if not q.is_cuda:
        hip._require_gpu(q)
    if not q.is_contiguous() or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_like(q)
    with _on(dev):
        hip.paged_shared_attention(q, k_pages, v_pages, out, block_table, plan, scale)
    return out


def default_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
