"""Tensor-level API over the C ABI: allocate outputs, derive strides and grids.

These are the calls a PyTorch user makes; each one is a single C-ABI call that
launches the sm_100a kernel on the current CUDA stream. Inputs must already be
CUDA tensors of the stated dtype; nothing is converted or copied implicitly
and there is no CPU path.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .kernels import current_stream_and_device


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, contiguous: bool = True) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device})")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def vector_add(x: torch.Tensor, y: torch.Tensor, out: torch.Tensor | None = None,
               block_size: int = 1024) -> torch.Tensor:
    """out = x + y over fp32 vectors (windows/kernels.py:7-15)."""
    _need(x, "x", torch.float32)
    _need(y, "y", torch.float32)
    if x.numel() != y.numel():
        raise ValueError("x and y must have the same number of elements")
    out = torch.empty_like(x) if out is None else out
    _need(out, "out", torch.float32)
    n = x.numel()
    stream = current_stream_and_device([x])
    _lib.call("neso_vector_add", x.data_ptr(), y.data_ptr(), out.data_ptr(), n, block_size,
              (n + block_size - 1) // block_size, 1, 1, stream)
    return out


def scale(x: torch.Tensor, factor: float, out: torch.Tensor | None = None, block_size: int = 1024) -> torch.Tensor:
    """out = x * factor over fp32 vectors (windows/kernels.py:18-22)."""
    _need(x, "x", torch.float32)
    out = torch.empty_like(x) if out is None else out
    _need(out, "out", torch.float32)
    n = x.numel()
    stream = current_stream_and_device([x])
    _lib.call("neso_scale", x.data_ptr(), out.data_ptr(), float(factor), n, block_size,
              (n + block_size - 1) // block_size, 1, 1, stream)
    return out


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None,
                    causal: bool = False, table: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """FA2 forward over contiguous fp16 [B, H, S, D] (D in {64, 128}); fp32 out.

    ``table`` (fp32 [H, 2S-1]) adds table[h, i - j + S - 1] to the logits.
    """
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, n, torch.float16)
    if q.dim() != 4 or q.shape != k.shape or q.shape != v.shape:
        raise ValueError("q, k, v must share one [B, H, S, D] shape")
    B, H, S, D = q.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device) if out is None else out
    _need(out, "out", torch.float32)
    stream = current_stream_and_device([q])
    if table is None:
        _lib.call("neso_fa2_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), B, H, S, D,
                  float(scale), int(bool(causal)), stream)
    else:
        _need(table, "table", torch.float32)
        if tuple(table.shape) != (H, 2 * S - 1):
            raise ValueError(f"table must be [H, 2S-1] = [{H}, {2 * S - 1}]")
        _lib.call("neso_fa2_fwd_relpos_table", q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(),
                  out.data_ptr(), B, H, S, D, float(scale), int(bool(causal)), stream)
    return out


def matmul(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """C (fp32) = A (fp16 [M, K]) @ B (fp16 [K, N]) (tests/test_aot.py:70-99)."""
    _need(a, "a", torch.float16)
    _need(b, "b", torch.float16)
    M, K = a.shape
    K2, N = b.shape
    if K != K2:
        raise ValueError("inner dimensions differ")
    out = torch.empty((M, N), dtype=torch.float32, device=a.device) if out is None else out
    _need(out, "out", torch.float32)
    stream = current_stream_and_device([a])
    _lib.call("neso_matmul_kernel", a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, K, 1, N, 1, N, 1,
              128, 128, 32, (M + 127) // 128, (N + 127) // 128, 1, stream)
    return out


def w8a16_matmul(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Y (fp32 [M, N]) = X (fp16 [M, K]) @ (W int8 [K, N] * scale fp16 [N])."""
    _need(x, "x", torch.float16)
    _need(w, "w", torch.int8)
    if scale is not None:
        _need(scale, "scale", torch.float16)
    M, K = x.shape
    N = w.shape[1]
    out = torch.empty((M, N), dtype=torch.float32, device=x.device) if out is None else out
    _need(out, "out", torch.float32)
    stream = current_stream_and_device([x])
    _lib.call("neso_w8a16_matmul_mnk", x.data_ptr(), w.data_ptr(), None if scale is None else scale.data_ptr(),
              out.data_ptr(), M, N, K, stream)
    return out


def pack_int4(q: torch.Tensor) -> torch.Tensor:
    """Pack int4 values q [K, N] in [-8, 7] (any integer dtype) into uint8
    [K/2, N]: byte (k/2, n) holds row k even in bits 0-3 and row k odd in bits
    4-7 (two's complement nibbles)."""
    if q.shape[0] % 2:
        raise ValueError("K must be even")
    u = (q.to(torch.int16) & 0xF).to(torch.uint8)
    return (u[0::2] | (u[1::2] << 4)).contiguous()


def w4a16_g128_matmul(x: torch.Tensor, wq: torch.Tensor, scales: torch.Tensor,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Y (fp32) = sum_g scales[g, n] * sum_{k in g} X[m, k] q[k, n] with packed
    int4 weights wq (uint8 [K/2, N]) and fp16 scales [K/128, N]."""
    _need(x, "x", torch.float16)
    _need(wq, "wq", torch.uint8)
    _need(scales, "scales", torch.float16)
    M, K = x.shape
    N = wq.shape[1]
    out = torch.empty((M, N), dtype=torch.float32, device=x.device) if out is None else out
    _need(out, "out", torch.float32)
    stream = current_stream_and_device([x])
    _lib.call("neso_w4a16_g128_matmul", x.data_ptr(), wq.data_ptr(), scales.data_ptr(), out.data_ptr(), M, N, K,
              stream)
    return out


# ------------------------------------------- one decoding step, paged cache --
#
# The cache is a pair of tensors [num_pages, Hkv, page_size, D] (fp16 or bf16;
# views with other strides are fine as long as D is contiguous and the rest are
# multiples of 8 elements). block_tables (int32 [B, width]) names the pages of
# each sequence, seq_lens (int32 [B]) its cached tokens. Lengths, tables,
# positions and slots stay on the device, so the calls can be captured in a
# CUDA graph and replayed with other values in them.

_binding = None


def _load_binding():
    """The extension module that checks and launches the operators below, with
    the library's entry points handed to it (once)."""
    global _binding
    if _binding is None:
        _binding = _lib.binding()
    return _binding


def rope_paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      positions: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      sections: list[int] | tuple[int, ...] | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q [N, Hq, D] and k [N, Hkv, D] of N new tokens, write k and v
    [N, Hkv, D] to the cache, and return the rotated q.

    cos, sin: fp32 [positions, half]; element pair (d, d + half), d < half,
    turns by the row of the token's position, elements from 2 * half on stay as
    they are. positions: int32 [N], or [axes, N] with ``sections`` (widths that
    add up to half): pair d takes the axis whose section holds it. slots: int64
    [N], page * page_size + row of each token; a slot outside the cache marks
    padding (not cached, its row of the result is zero); the others must
    differ. A position outside the table gives NaN. ``out`` may be q."""
    return (_binding or _load_binding()).rope_paged_append(q, k, v, cos, sin, positions, slots, k_cache, v_cache, sections, out)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float | None = None, softcap: float = 0.0, window: int = 0,
                    slopes: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                    weights_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its cached tokens (the new
    one included); q [B, Hq, D] (D in {64, 128}), result [B, Hq, D] in q's type.

    ``softcap`` > 0 caps the scaled scores s as softcap * tanh(s / softcap),
    ``slopes`` (fp32 [Hq]) then adds slope * (t - (len - 1)), ``window`` > 0
    keeps the last ``window`` tokens. ``weights`` (fp32 [B, Hkv, tokens], tokens
    at least width * page_size) has the softmax weights of each kv head's
    query heads added, in place or into ``weights_out``, for t < len.

    Lengths are clamped to [0, width * page_size]; tokens of a page outside the
    cache are left out; a sequence without tokens gives zeros. ``slopes`` and
    ``window`` count cached tokens: after ``kv_evict`` these are distances in the
    trimmed cache, not between the positions that the keys were rotated by."""
    return (_binding or _load_binding()).paged_attention(q, k_cache, v_cache, block_tables, seq_lens, scale, softcap, window,
                                                       slopes, weights, weights_out, out)


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
             weights: torch.Tensor, budget: int, recent: int, sink: int = 0,
             out_tables: torch.Tensor | None = None,
             weights_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Trim every sequence to ``budget`` (1 to 2^30) tokens per kv head: the first ``sink``,
    the last ``recent`` and the ones with the largest ``weights`` (fp32 [B, Hkv,
    tokens], tokens at least width * page_size, as ``paged_attention``
    accumulates them) between. Kept tokens stay
    in order and move to the sequence's first slots under ``out_tables`` (int32
    [B, width]; None: in place, under block_tables), their weights to the front
    of ``weights_out`` (None: in place), followed by zeros up to the old length.
    Returns the kept tokens' old indexes (int32 [B, Hkv, budget], -1 behind the
    last) and the new lengths (int32 [B]).

    ``out_tables`` is block_tables itself or a view of its first columns (in
    place), or a table of its own whose pages either lie where block_tables has
    them or do not occur in it. A sequence with pages that stay, as under a copy
    of block_tables, moves in order and more slowly than in place. No page may
    belong to two sequences."""
    return (_binding or _load_binding()).kv_evict(k_cache, v_cache, block_tables, seq_lens, weights, budget, recent, sink,
                                                out_tables, weights_out)


def process_logits(logits: torch.Tensor, history: torch.Tensor | None = None,
                   history_lens: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                   repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                   presence: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties, biases and a grammar mask on logits [B, V] (fp32, fp16 or
    bf16; computed in fp32, rounded once).

    history (int32 [B, T]) holds history_lens[b] token ids, the first
    prompt_lens[b] of them the prompt. A token of the history has x divided by
    repetition[b] if positive, else multiplied by it; one generated n > 0 times
    has frequency[b] * n + presence[b] subtracted. bias (fp32 [B, n]) is added
    at bias_ids (int32 [B, n]; ids outside the vocabulary, -1 for instance,
    are skipped). mask (int32 [B, ceil(V / 32)]): bit v % 32 of word v / 32
    allows token v, the others become -inf. ``out`` may be logits."""
    return (_binding or _load_binding()).process_logits(logits, history, history_lens, prompt_lens, repetition, frequency,
                                                      presence, bias_ids, bias, mask, out)
