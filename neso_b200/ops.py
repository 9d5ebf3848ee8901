"""Tensor-level API over the C ABI: allocate outputs, derive strides and grids.

These are the calls a PyTorch user makes; each one is a single C-ABI call that
launches the sm_100a kernel on the current CUDA stream. Inputs must already be
CUDA tensors of the stated dtype; nothing is converted or copied implicitly
and there is no CPU path.
"""
from __future__ import annotations

import ctypes
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

_DTYPES = {torch.float16: _lib.NESO_F16, torch.bfloat16: _lib.NESO_BF16, torch.float32: _lib.NESO_F32}


def _tensor(t: torch.Tensor, name: str, dtypes: tuple, dim: int, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device})")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(map(str, dtypes))} (got {t.dtype})")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions (got {t.dim()})")
    return t


def _rows(t: torch.Tensor, name: str) -> None:
    """The last dimension has to be contiguous (a length of one always is)."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _stride(t: torch.Tensor, dim: int) -> int:
    """Stride of a dimension; 0 where its length leaves the stride without a meaning."""
    return t.stride(dim) if t.shape[dim] > 1 else 0


def _written(t: torch.Tensor, name: str) -> None:
    if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"{name} is written to and must not be an expanded view")


def _extent(t: torch.Tensor) -> tuple[int, int]:
    first = t.data_ptr()
    if t.numel() == 0:
        return first, first
    return first, first + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _same_or_apart(a: torch.Tensor, b: torch.Tensor, what: str) -> None:
    """An output may be the input itself or must not touch it."""
    a0, a1 = _extent(a)
    b0, b1 = _extent(b)
    if a0 < b1 and b0 < a1 and not (a0 == b0 and a.shape == b.shape and a.stride() == b.stride()):
        raise ValueError(f"{what} overlap without being the same tensor")


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, device: torch.device) -> tuple[int, int, int, int]:
    _tensor(k_cache, "k_cache", (torch.float16, torch.bfloat16), 4, device)
    _tensor(v_cache, "v_cache", (k_cache.dtype,), 4, device)
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must share one [num_pages, Hkv, page_size, D] shape")
    _rows(k_cache, "k_cache")
    _rows(v_cache, "v_cache")
    return tuple(k_cache.shape)


def _cache_strides(t: torch.Tensor) -> tuple[int, int, int]:
    return _stride(t, 0), _stride(t, 1), _stride(t, 2)


def _tables(block_tables: torch.Tensor, name: str, batch: int, device: torch.device) -> None:
    _tensor(block_tables, name, (torch.int32,), 2, device)
    _rows(block_tables, name)
    if block_tables.shape[0] != batch:
        raise ValueError(f"{name} must have one row per sequence ({batch})")


def _vector(t: torch.Tensor, name: str, dtype: torch.dtype, n: int, device: torch.device) -> None:
    _tensor(t, name, (dtype,), 1, device)
    _rows(t, name)
    if t.shape[0] != n:
        raise ValueError(f"{name} must have {n} elements (got {t.shape[0]})")


def _weights(t: torch.Tensor, name: str, batch: int, hkv: int, capacity: int, device: torch.device) -> None:
    _tensor(t, name, (torch.float32,), 3, device)
    _rows(t, name)
    if t.shape[0] != batch or t.shape[1] != hkv or t.shape[2] < capacity:
        raise ValueError(f"{name} must be [{batch}, {hkv}, at least {capacity} tokens] (got {list(t.shape)})")


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
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    device = q.device
    _tensor(q, "q", (torch.float16, torch.bfloat16), 3, device)
    pages, hkv, page_size, D = _caches(k_cache, v_cache, device)
    N, hq = q.shape[0], q.shape[1]
    for t, name in ((k, "k"), (v, "v")):
        _tensor(t, name, (q.dtype,), 3, device)
        if tuple(t.shape) != (N, hkv, D):
            raise ValueError(f"{name} must be [{N}, {hkv}, {D}] (got {list(t.shape)})")
    if q.shape[2] != D or k_cache.dtype != q.dtype:
        raise ValueError("q and the cache must share one head_dim and dtype")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _rows(t, name)
    for t, name in ((cos, "cos"), (sin, "sin")):
        _tensor(t, name, (torch.float32,), 2, device)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if cos.shape != sin.shape:
        raise ValueError("cos and sin must share one shape")
    half = cos.shape[1]
    _tensor(positions, "positions", (torch.int32,), 1 if isinstance(positions, torch.Tensor) and positions.dim() == 1 else 2,
            device)
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    if positions.shape[-1] != N or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous [{N}] or [axes, {N}]")
    if sections is None:
        if axes != 1:
            raise ValueError("several position axes need sections")
        widths = None
    else:
        if len(sections) != axes:
            raise ValueError(f"sections must have one width per axis ({axes})")
        widths = (ctypes.c_int32 * axes)(*sections)
    _vector(slots, "slots", torch.int64, N, device)
    _written(k_cache, "k_cache")
    _written(v_cache, "v_cache")
    if out is None:
        out = torch.empty((N, hq, D), dtype=q.dtype, device=device)
    else:
        _tensor(out, "out", (q.dtype,), 3, device)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and of q's shape")
        _same_or_apart(out, q, "out and q")
    stream = current_stream_and_device([q])
    _lib.call("neso_rope_paged_append", q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(),
              positions.data_ptr(), slots.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
              _DTYPES[q.dtype], N, hq, hkv, D, half, cos.shape[0], axes, widths, _stride(q, 0), _stride(q, 1),
              _stride(k, 0), _stride(k, 1), _stride(v, 0), _stride(v, 1), pages, page_size, *_cache_strides(k_cache),
              *_cache_strides(v_cache), stream)
    return out


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
    cache are left out; a sequence without tokens gives zeros."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    device = q.device
    _tensor(q, "q", (torch.float16, torch.bfloat16), 3, device)
    _rows(q, "q")
    pages, hkv, page_size, D = _caches(k_cache, v_cache, device)
    B, hq = q.shape[0], q.shape[1]
    if q.shape[2] != D or k_cache.dtype != q.dtype:
        raise ValueError("q and the cache must share one head_dim and dtype")
    _tables(block_tables, "block_tables", B, device)
    _vector(seq_lens, "seq_lens", torch.int32, B, device)
    width = block_tables.shape[1]
    if slopes is not None:
        _vector(slopes, "slopes", torch.float32, hq, device)
    win_s = wout_s = (0, 0)
    if weights is not None:
        _weights(weights, "weights", B, hkv, width * page_size, device)
        if weights_out is None:
            weights_out = weights
        else:
            _weights(weights_out, "weights_out", B, hkv, width * page_size, device)
            _same_or_apart(weights_out, weights, "weights and weights_out")
        _written(weights_out, "weights_out")
        win_s = (_stride(weights, 0), _stride(weights, 1))
        wout_s = (_stride(weights_out, 0), _stride(weights_out, 1))
    elif weights_out is not None:
        raise ValueError("weights_out needs weights")
    if out is None:
        out = torch.empty((B, hq, D), dtype=q.dtype, device=device)
    else:
        _tensor(out, "out", (q.dtype,), 3, device)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and of q's shape")
        a, b = _extent(out), _extent(q)
        if a[0] < b[1] and b[0] < a[1]:
            raise ValueError("out must not overlap q")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    stream = current_stream_and_device([q])
    need = _lib.lib().neso_paged_attention_workspace(B, hq, hkv, D, width, page_size, int(weights is not None))
    if need < 0:
        _lib.check(need, "neso_paged_attention")
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.call("neso_paged_attention", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(),
              seq_lens.data_ptr(), None if slopes is None else slopes.data_ptr(),
              None if weights is None else weights.data_ptr(), None if weights is None else weights_out.data_ptr(),
              out.data_ptr(), workspace.data_ptr(), need, _DTYPES[q.dtype], B, hq, hkv, D, float(scale),
              float(softcap), window, _stride(q, 0), _stride(q, 1), pages, page_size, *_cache_strides(k_cache),
              *_cache_strides(v_cache), width, _stride(block_tables, 0), *win_s, *wout_s, stream)
    return out


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
             weights: torch.Tensor, budget: int, recent: int, sink: int = 0,
             out_tables: torch.Tensor | None = None,
             weights_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Trim every sequence to ``budget`` tokens per kv head: the first ``sink``,
    the last ``recent`` and the ones with the largest ``weights`` (fp32 [B, Hkv,
    tokens], as ``paged_attention`` accumulates them) between. Kept tokens stay
    in order and move to the sequence's first slots under ``out_tables`` (int32
    [B, width]; None: in place, under block_tables), their weights to the front
    of ``weights_out`` (None: in place), followed by zeros up to the old length.
    Returns the kept tokens' old indexes (int32 [B, Hkv, budget], -1 behind the
    last) and the new lengths (int32 [B]).

    Pages of ``out_tables`` must be other than every page of block_tables,
    unless the table is the same; no page may belong to two sequences."""
    if not isinstance(k_cache, torch.Tensor):
        raise TypeError("k_cache must be a torch.Tensor")
    device = k_cache.device
    pages, hkv, page_size, D = _caches(k_cache, v_cache, device)
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        raise ValueError("block_tables must be a [B, width] tensor")
    B, width = block_tables.shape
    _tables(block_tables, "block_tables", B, device)
    _vector(seq_lens, "seq_lens", torch.int32, B, device)
    _weights(weights, "weights", B, hkv, width * page_size, device)
    if weights_out is None:
        weights_out = weights
    else:
        _weights(weights_out, "weights_out", B, hkv, width * page_size, device)
        _same_or_apart(weights_out, weights, "weights and weights_out")
    if out_tables is None:
        out_tables = block_tables
    else:
        _tables(out_tables, "out_tables", B, device)
        if out_tables.shape[1] * page_size < min(budget, width * page_size):
            raise ValueError(f"out_tables hold {out_tables.shape[1] * page_size} tokens per sequence, "
                             f"{min(budget, width * page_size)} may be kept")
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache"), (weights_out, "weights_out")):
        _written(t, name)
    kept = torch.empty((B, hkv, max(budget, 0)), dtype=torch.int32, device=device)
    new_lens = torch.empty(B, dtype=torch.int32, device=device)
    stream = current_stream_and_device([k_cache])
    _lib.call("neso_kv_evict", k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), out_tables.data_ptr(),
              seq_lens.data_ptr(), weights.data_ptr(), weights_out.data_ptr(), kept.data_ptr(), new_lens.data_ptr(),
              B, hkv, D, budget, recent, sink, pages, page_size, *_cache_strides(k_cache), *_cache_strides(v_cache),
              width, _stride(block_tables, 0), out_tables.shape[1], _stride(out_tables, 0), _stride(weights, 0),
              _stride(weights, 1), _stride(weights_out, 0), _stride(weights_out, 1), stream)
    return kept, new_lens


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
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    device = logits.device
    _tensor(logits, "logits", (torch.float32, torch.float16, torch.bfloat16), 2, device)
    _rows(logits, "logits")
    B, V = logits.shape
    T = 0
    if history is not None:
        _tensor(history, "history", (torch.int32,), 2, device)
        _rows(history, "history")
        if history.shape[0] != B or history_lens is None:
            raise ValueError(f"history must have one row per sequence ({B}) and come with history_lens")
        T = history.shape[1]
        _vector(history_lens, "history_lens", torch.int32, B, device)
        if prompt_lens is not None:
            _vector(prompt_lens, "prompt_lens", torch.int32, B, device)
    elif history_lens is not None or prompt_lens is not None:
        raise ValueError("history_lens and prompt_lens need a history")
    for t, name in ((repetition, "repetition"), (frequency, "frequency"), (presence, "presence")):
        if t is not None:
            _vector(t, name, torch.float32, B, device)
            if history is None:
                raise ValueError(f"{name} needs a history")
    n_bias = 0
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias come together")
    if bias is not None:
        _tensor(bias_ids, "bias_ids", (torch.int32,), 2, device)
        _tensor(bias, "bias", (torch.float32,), 2, device)
        n_bias = bias.shape[1]
        if bias.shape != bias_ids.shape or bias.shape[0] != B or not (bias.is_contiguous() and bias_ids.is_contiguous()):
            raise ValueError(f"bias_ids and bias must be contiguous and share one [{B}, n] shape")
    if mask is not None:
        _tensor(mask, "mask", (torch.int32,), 2, device)
        _rows(mask, "mask")
        if mask.shape[0] != B or mask.shape[1] < (V + 31) // 32:
            raise ValueError(f"mask must be [{B}, at least {(V + 31) // 32} words]")
    if out is None:
        out = torch.empty((B, V), dtype=logits.dtype, device=device)
    else:
        _tensor(out, "out", (logits.dtype,), 2, device)
        _rows(out, "out")
        if out.shape != logits.shape:
            raise ValueError("out must have the shape of logits")
        _same_or_apart(out, logits, "out and logits")
        _written(out, "out")
    stream = current_stream_and_device([logits])

    def ptr(t):
        return None if t is None else t.data_ptr()

    _lib.call("neso_process_logits", logits.data_ptr(), out.data_ptr(), _DTYPES[logits.dtype], B, V,
              _stride(logits, 0), _stride(out, 0), ptr(history), ptr(history_lens), ptr(prompt_lens), T,
              0 if history is None else _stride(history, 0), ptr(repetition), ptr(frequency), ptr(presence),
              ptr(bias_ids), ptr(bias), n_bias, ptr(mask), 0 if mask is None else _stride(mask, 0), stream)
    return out
