"""Torch CPU float64 statements of the decoding-step operators — TEST INFRASTRUCTURE ONLY.

Each function is the operator's definition written out per sequence and head,
in 64 bits, on CPU tensors; nothing is shared with the kernels' layout of the
work. Caches are [num_pages, Hkv, page_size, D] tensors.
"""
from __future__ import annotations

import math

import torch

__all__ = ["decode_rope", "decode_rows", "decode_attention", "decode_evict", "decode_logits"]


def decode_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                sections: list[int]) -> torch.Tensor:
    """x [N, H, D] rotated in 64 bits; positions [axes, N]; a position outside the table gives NaN."""
    half = cos.shape[1]
    y = x.double().clone()
    axis = [a for a, w in enumerate(sections) for _ in range(w)]
    for n in range(x.shape[0]):
        for d in range(half):
            p = int(positions[axis[d], n])
            c, s = (float(cos[p, d]), float(sin[p, d])) if 0 <= p < cos.shape[0] else (math.nan, math.nan)
            a, b = x[n, :, d].double(), x[n, :, d + half].double()
            y[n, :, d] = a * c - b * s
            y[n, :, d + half] = a * s + b * c
    return y


def decode_rows(cache: torch.Tensor, table: torch.Tensor, tokens: list[int], head: int) -> torch.Tensor:
    """Rows of the given tokens of one sequence and kv head, [tokens, D]."""
    page = cache.shape[2]
    return torch.stack([cache[int(table[t // page]), head, t % page] for t in tokens])


def decode_attention(q, k_cache, v_cache, tables, lens, scale, softcap=0.0, window=0, slopes=None):
    """Returns (out [B, Hq, D], weight sums {(b, kv): {t: sum}}, bounds) where
    bounds [B, Hq, 2] holds, for the visible tokens of a row, the largest
    sum_d |q_d k_d| * |scale| and the sum of p |v| over its largest element."""
    B, hq, D = q.shape
    hkv, page, pages = k_cache.shape[1], k_cache.shape[2], k_cache.shape[0]
    group = hq // hkv
    out = torch.zeros(B, hq, D, dtype=torch.float64)
    bounds = torch.zeros(B, hq, 2, dtype=torch.float64)
    sums = {}
    for b in range(B):
        n = min(max(int(lens[b]), 0), tables.shape[1] * page)
        lo = max(0, n - window) if window else 0
        toks = [t for t in range(lo, n) if 0 <= int(tables[b, t // page]) < pages]
        for kv in range(hkv):
            if not toks:
                continue
            k = decode_rows(k_cache, tables[b], toks, kv).double()
            v = decode_rows(v_cache, tables[b], toks, kv).double()
            total = torch.zeros(len(toks), dtype=torch.float64)
            for h in range(kv * group, (kv + 1) * group):
                s = (k @ q[b, h].double()) * scale
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    s = s + float(slopes[h]) * (torch.tensor(toks, dtype=torch.float64) - (n - 1))
                p = torch.exp(s - s.max())
                p = p / p.sum()
                out[b, h] = p @ v
                total += p
                bounds[b, h, 0] = ((k.abs() @ q[b, h].double().abs()) * abs(scale)).max()
                bounds[b, h, 1] = (p @ v.abs()).max()
            sums[b, kv] = dict(zip(toks, total.tolist()))
    return out, sums, bounds


def decode_evict(weights, lens, budget, recent, sink, capacity):
    """kept[b][kv]: the kept tokens, ascending. NaN ranks above everything."""
    kept = []
    for b in range(weights.shape[0]):
        n = min(max(int(lens[b]), 0), capacity)
        rows = []
        for kv in range(weights.shape[1]):
            if n <= budget:
                rows.append(list(range(n)))
                continue
            w = weights[b, kv].tolist()
            middle = range(sink, n - recent)
            order = sorted(middle, key=lambda t: (-math.inf if math.isnan(w[t]) else -w[t], not math.isnan(w[t]), t))
            best = order[:budget - sink - recent]
            rows.append(sorted(list(range(sink)) + best + list(range(n - recent, n))))
        kept.append(rows)
    return kept


def decode_logits(logits, history=None, history_lens=None, prompt_lens=None, repetition=None, frequency=None,
                  presence=None, bias_ids=None, bias=None, mask=None):
    """Returns (values [B, V], magnitude [B, V]): the magnitude sums the absolute
    values of everything that was added or scaled on the way."""
    x = logits.double().clone()
    mag = x.abs()
    B, V = x.shape
    for b in range(B):
        ids, made = [], []
        if history is not None:
            n = min(max(int(history_lens[b]), 0), history.shape[1])
            first = int(prompt_lens[b]) if prompt_lens is not None else 0
            row = history[b].tolist()
            ids = [t for t in row[:n] if 0 <= t < V]
            made = [t for i, t in enumerate(row[:n]) if 0 <= t < V and i >= first]
        for t in set(ids):
            r = float(repetition[b]) if repetition is not None else 1.0
            x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
            mag[b, t] = x[b, t].abs()
        for t in set(made):
            c = made.count(t)
            f = float(frequency[b]) * c if frequency is not None else 0.0
            p = float(presence[b]) if presence is not None else 0.0
            x[b, t] -= f + p
            mag[b, t] += abs(f) + abs(p)
        if bias is not None:
            for t, v in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= t < V:
                    x[b, t] += v
                    mag[b, t] += abs(v)
        if mask is not None:
            for t in range(V):
                if not (int(mask[b, t // 32]) >> (t % 32)) & 1:
                    x[b, t] = -math.inf
    return x, mag
