"""The operators of one decoding step over a paged key-value cache, as cases to measure.

Four operators, in the order in which a serving loop calls them:

* ``append``  rotates the queries and keys of new tokens (one or several position axes) and writes
  keys and values into the pages of the cache;
* ``attend``  attention of one new token per sequence over its pages, optionally adding the
  weights that each cached token received to a running sum;
* ``evict``   keeps the tokens with the largest accumulated weight and moves them together;
* ``logits``  penalties for repeated tokens, sparse biases and a grammar mask on the next token's logits.

``own`` selects what ``run`` calls: the plain torch form (False) or this framework's kernels (True).
"""
import math
import random

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one sequence decoding, one position axis: launch latency is all there is
        dict(name="append_token", op="append", dtype="f16", tokens=1, hq=16, hkv=16, d=64, half=32, axes=1, page=16,
             table=4096, fused=True),
        # a batch of decoding sequences, odd count, part of the head rotated
        dict(name="append_batch", op="append", dtype="bf16", tokens=187, hq=32, hkv=8, d=128, half=32, axes=1, page=32,
             table=8192, fused=True),
        # prompts of image and video tokens: three axes (time, height, width), views of one fused projection
        dict(name="append_prompt", op="append", dtype="bf16", tokens=8192, hq=32, hkv=8, d=128, half=64, axes=3,
             page=16, table=16384, fused=True),
        # the first tokens of one chat: one short sequence, one query head per key head
        dict(name="attend_short", op="attend", dtype="f16", batch=1, hq=16, hkv=16, d=64, page=16, lo=129, hi=129,
             softcap=0.0, window=0, alibi=False, weights=False, lens_seed=1),
        # one very long document, grouped heads: the split over the cache's length carries it
        dict(name="attend_long", op="attend", dtype="bf16", batch=1, hq=32, hkv=8, d=128, page=16, lo=131071, hi=131071,
             softcap=0.0, window=0, alibi=False, weights=False, lens_seed=2),
        # a busy server: ragged lengths from a few tokens to thousands
        dict(name="attend_ragged", op="attend", dtype="f16", batch=64, hq=64, hkv=8, d=128, page=16, lo=5, hi=8192,
             softcap=0.0, window=0, alibi=False, weights=False, lens_seed=3),
        # capped scores, a distance bias and a sliding window, odd group and page sizes
        dict(name="attend_window", op="attend", dtype="bf16", batch=48, hq=24, hkv=8, d=64, page=24, lo=300, hi=6000,
             softcap=30.0, window=1025, alibi=True, weights=False, lens_seed=4),
        # a budgeted cache: the weights of every cached token are accumulated for the eviction
        dict(name="attend_weights", op="attend", dtype="f16", batch=16, hq=32, hkv=8, d=128, page=64, lo=2049, hi=4096,
             softcap=0.0, window=0, alibi=False, weights=True, lens_seed=5),
        # one sequence trimmed to half its pages
        dict(name="evict_one", op="evict", dtype="f16", batch=1, hkv=8, d=64, page=16, lo=1023, hi=1023, budget=512,
             recent=32, sink=4, lens_seed=6),
        # a batch trimmed after its prompts
        dict(name="evict_batch", op="evict", dtype="bf16", batch=8, hkv=8, d=128, page=32, lo=1800, hi=4096, budget=2048,
             recent=256, sink=4, lens_seed=7),
        # one row of logits, a short history, no grammar
        dict(name="logits_row", op="logits", dtype="f32", batch=1, vocab=32000, history=300, bias=0, mask=False,
             lens_seed=8),
        # a batch under a grammar with long histories and odd vocabulary
        dict(name="logits_grammar", op="logits", dtype="f32", batch=128, vocab=128257, history=4096, bias=16, mask=True,
             lens_seed=9),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "logits"])
    seed = rng.randrange(1 << 20)
    if op == "append":
        d = rng.choice([64, 128])
        hkv = rng.choice([1, 2, 4, 8, 16])
        axes = rng.choice([1, 1, 2, 3])
        return dict(op=op, dtype=rng.choice(["f16", "bf16"]), tokens=_log(rng, 1, 8192),
                    hq=hkv * rng.choice([1, 2, 3, 4]) if hkv > 4 else hkv * rng.choice([1, 4, 6, 8]), hkv=hkv, d=d,
                    half=rng.choice([d // 2, d // 2, d // 4, 24]), axes=axes, page=rng.choice([8, 16, 24, 64, 128]),
                    table=_log(rng, 1024, 32768), fused=rng.random() < 0.5)
    if op == "attend":
        d = rng.choice([64, 128])
        hkv = rng.choice([1, 2, 4, 8, 16])
        batch = _log(rng, 1, 128)
        hi = _log(rng, 1, 131072)
        while batch * hi * hkv * d > 131072 * 8 * 128:
            hi = max(1, hi // 2)
        weights = rng.random() < 0.3 and batch * hi * hkv <= 1 << 20
        return dict(op=op, dtype=rng.choice(["f16", "bf16"]), batch=batch, hq=hkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16]),
                    hkv=hkv, d=d, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256]), lo=max(1, hi // rng.choice([1, 2, 50])),
                    hi=hi, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
                    alibi=rng.random() < 0.25, weights=weights, lens_seed=seed)
    if op == "evict":
        hkv = rng.choice([1, 2, 4, 8])
        batch = _log(rng, 1, 32)
        hi = _log(rng, 64, 16384)
        while batch * hi * hkv > 8 * 8 * 4096:
            hi //= 2
        budget = max(1, int(hi * rng.uniform(0.2, 0.8)))
        recent = rng.randrange(0, budget // 2 + 1)
        return dict(op=op, dtype=rng.choice(["f16", "bf16"]), batch=batch, hkv=hkv, d=rng.choice([64, 128]),
                    page=rng.choice([8, 16, 24, 64, 128]), lo=max(1, hi // rng.choice([1, 2, 4])), hi=hi, budget=budget,
                    recent=recent, sink=rng.randrange(0, min(8, budget - recent) + 1), lens_seed=seed)
    batch = _log(rng, 1, 128)
    vocab = _log(rng, 1000, 128257)
    return dict(op=op, dtype=rng.choice(["f16", "bf16", "f32"]), batch=batch, vocab=vocab, history=_log(rng, 1, 4096),
                bias=rng.choice([0, 1, 7, 32]), mask=rng.random() < 0.5, lens_seed=seed)


def _lens(case):
    rng = random.Random(case["lens_seed"])
    n = case["batch"]
    lo, hi = case["lo"], case["hi"]
    lens = [hi] + [_log(rng, lo, hi) for _ in range(n - 1)]
    rng.shuffle(lens)
    return lens


def _history_lens(case):
    rng = random.Random(case["lens_seed"])
    lens = [case["history"]] + [rng.randrange(0, case["history"] + 1) for _ in range(case["batch"] - 1)]
    return lens, [rng.randrange(0, n + 1) for n in lens]


# ----------------------------------------------------------------- inputs --
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"append": _prepare_append, "attend": _prepare_attend, "evict": _prepare_evict,
            "logits": _prepare_logits}[case["op"]](case, g)


def _normal(shape, dtype, g, scale=1.0):
    x = torch.randn(shape, device="cuda", generator=g)
    return x.mul_(scale).to(dtype) if scale != 1.0 else x.to(dtype)


def _sections(half, axes):
    # time gets the remainder, as the slowest axis
    rest = half // (axes + 1) if axes > 1 else 0
    return [half - rest * (axes - 1)] + [rest] * (axes - 1)


def _prepare_append(case, g):
    n, hq, hkv, d, half = (case[k] for k in ("tokens", "hq", "hkv", "d", "half"))
    dt = _DT[case["dtype"]]
    if case["fused"]:
        qkv = _normal((n, hq + 2 * hkv, d), dt, g)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    else:
        q, k, v = (_normal((n, h, d), dt, g) for h in (hq, hkv, hkv))
    pos = torch.arange(case["table"], device="cuda", dtype=torch.float64)
    freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = pos[:, None] * freq
    pages = -(-n // case["page"]) + 3
    slots = torch.randperm(pages * case["page"], device="cuda", generator=g)[:n]
    positions = torch.randint(0, case["table"], (case["axes"], n), device="cuda", generator=g, dtype=torch.int32)
    kc, vc = (_normal((pages, hkv, case["page"], d), dt, g) for _ in range(2))
    return dict(case=case, q=q, k=k, v=v, cos=angle.cos().float(), sin=angle.sin().float(), positions=positions,
                slots=slots, k_cache=kc, v_cache=vc, sections=_sections(half, case["axes"]))


def _tables(lens, page, g, first=0):
    """Block tables over pages in a shuffled order, each sequence with pages of its own."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), device="cuda", generator=g).to(torch.int32) + first
    table = torch.zeros((len(lens), max(max(need), 1)), device="cuda", dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    return table, sum(need)


def _prepare_attend(case, g):
    dt = _DT[case["dtype"]]
    lens = _lens(case)
    b, hq, hkv, d = (case[k] for k in ("batch", "hq", "hkv", "d"))
    table, pages = _tables(lens, case["page"], g)
    st = dict(case=case, lens=lens, q=_normal((b, hq, d), dt, g, 2.0), table=table,
              k_cache=_normal((pages, hkv, case["page"], d), dt, g), v_cache=_normal((pages, hkv, case["page"], d), dt, g),
              seq_lens=torch.tensor(lens, device="cuda", dtype=torch.int32), slopes=None, weights=None)
    if case["alibi"]:
        st["slopes"] = torch.rand(hq, device="cuda", generator=g) * 0.05
    if case["weights"]:
        st["weights"] = torch.rand((b, hkv, table.shape[1] * case["page"]), device="cuda", generator=g)
        st["weights_out"] = st["weights"].clone()
    return st


def _prepare_evict(case, g):
    dt = _DT[case["dtype"]]
    lens = _lens(case)
    b, hkv, d, page = (case[k] for k in ("batch", "hkv", "d", "page"))
    table, pages = _tables(lens, page, g)
    keep = [min(n, case["budget"]) for n in lens]
    out_table, more = _tables(keep, page, g, first=pages)
    shape = (pages + more, hkv, page, d)
    w = torch.rand((b, hkv, table.shape[1] * page), device="cuda", generator=g)
    # most tokens get little weight, some none at all: those tie
    w = torch.where(w < 0.1, torch.zeros_like(w), w.pow(8) * 50.0)
    return dict(case=case, lens=lens, table=table, out_table=out_table, k_cache=_normal(shape, dt, g),
                v_cache=_normal(shape, dt, g), seq_lens=torch.tensor(lens, device="cuda", dtype=torch.int32), weights=w,
                weights_out=torch.zeros_like(w))


def _prepare_logits(case, g):
    b, v, t = case["batch"], case["vocab"], case["history"]
    lens, prompt = _history_lens(case)
    logits = _normal((b, v), _DT[case["dtype"]], g, 4.0)
    # token ids fall off like word frequencies, so many repeat
    ids = (torch.rand((b, t), device="cuda", generator=g).pow(4) * v).to(torch.int32).clamp_(max=v - 1)
    st = dict(case=case, logits=logits, history=ids, history_lens=torch.tensor(lens, device="cuda", dtype=torch.int32),
              prompt_lens=torch.tensor(prompt, device="cuda", dtype=torch.int32),
              repetition=1.0 + 0.3 * torch.rand(b, device="cuda", generator=g),
              frequency=0.5 * torch.rand(b, device="cuda", generator=g),
              presence=torch.rand(b, device="cuda", generator=g), bias_ids=None, bias=None, mask=None)
    if case["bias"]:
        step = v // case["bias"]
        base = torch.arange(case["bias"], device="cuda", dtype=torch.int32) * step
        st["bias_ids"] = base + torch.randint(0, step, (b, case["bias"]), device="cuda", generator=g, dtype=torch.int32)
        st["bias"] = torch.randn((b, case["bias"]), device="cuda", generator=g) * 5.0
    if case["mask"]:
        words = -(-v // 32)
        mask = torch.randint(-(1 << 31), 1 << 31, (b, words), device="cuda", generator=g).to(torch.int32)
        mask &= torch.randint(-(1 << 31), 1 << 31, (b, words), device="cuda", generator=g).to(torch.int32)
        mask[::7] = -1   # rows without a grammar
        mask[3::16] = 0  # a grammar that has come to its end
        st["mask"] = mask
    return st


# -------------------------------------------------------------------- run --
def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "evict": _own_evict, "logits": _own_logits}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "logits": _plain_logits}[op](state)


def _own_append(st):
    from neso_b200 import ops
    q = ops.rope_paged_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["positions"], st["slots"],
                              st["k_cache"], st["v_cache"], sections=st["sections"])
    return q, st["k_cache"], st["v_cache"]


def _own_attend(st):
    from neso_b200 import ops
    c = st["case"]
    out = ops.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["seq_lens"], softcap=c["softcap"],
                              window=c["window"], slopes=st["slopes"], weights=st["weights"],
                              weights_out=st["weights_out"] if c["weights"] else None)
    return (out, st["weights_out"]) if c["weights"] else out


def _own_evict(st):
    from neso_b200 import ops
    c = st["case"]
    kept, lens = ops.kv_evict(st["k_cache"], st["v_cache"], st["table"], st["seq_lens"], st["weights"], c["budget"],
                              c["recent"], sink=c["sink"], out_tables=st["out_table"], weights_out=st["weights_out"])
    return kept, lens, st["weights_out"], st["k_cache"], st["v_cache"]


def _own_logits(st):
    from neso_b200 import ops
    return ops.process_logits(st["logits"], history=st["history"], history_lens=st["history_lens"],
                              prompt_lens=st["prompt_lens"], repetition=st["repetition"], frequency=st["frequency"],
                              presence=st["presence"], bias_ids=st["bias_ids"], bias=st["bias"], mask=st["mask"])


def _plain_append(st):
    page = st["case"]["page"]
    axis = torch.repeat_interleave(torch.arange(len(st["sections"]), device="cuda"),
                                   torch.tensor(st["sections"], device="cuda"), output_size=st["cos"].shape[1])
    row = st["positions"][axis].long().t()
    col = torch.arange(st["cos"].shape[1], device="cuda")
    cos, sin = st["cos"][row, col][:, None], st["sin"][row, col][:, None]
    half = col.numel()

    def rotate(x):
        x = x.float()
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]], -1).to(st["q"].dtype)

    block, at = st["slots"] // page, st["slots"] % page
    st["k_cache"][block, :, at] = rotate(st["k"])
    st["v_cache"][block, :, at] = st["v"]
    return rotate(st["q"]), st["k_cache"], st["v_cache"]


def _gather(cache, table, n, start=0):
    """Tokens start..n-1 of one sequence as [kv heads, tokens, d]."""
    page = cache.shape[2]
    first = start // page
    rows = cache[table[first:-(-n // page)].long()].transpose(0, 1).flatten(1, 2)
    return rows[:, start - first * page:n - first * page]


def _plain_attend(st):
    c = st["case"]
    hkv, d = c["hkv"], c["d"]
    group = c["hq"] // hkv
    out = torch.empty_like(st["q"])
    wout = st["weights_out"] if c["weights"] else None
    for b, n in enumerate(st["lens"]):
        start = max(0, n - c["window"]) if c["window"] else 0
        k, v = (_gather(st[x], st["table"][b], n, start).float() for x in ("k_cache", "v_cache"))
        s = torch.matmul(st["q"][b].float().view(hkv, group, d), k.transpose(1, 2)) * (1.0 / math.sqrt(d))
        if c["softcap"]:
            s = c["softcap"] * torch.tanh(s / c["softcap"])
        if c["alibi"]:
            s = s + st["slopes"].view(hkv, group, 1) * torch.arange(start - n + 1, 1, device="cuda")
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out[b] = torch.matmul(p, v).view(-1, d).to(out.dtype)
        if c["weights"]:
            wout[b, :, :n] = st["weights"][b, :, :n]
            wout[b, :, start:n] += p.sum(1)
    return (out, wout) if c["weights"] else out


def _plain_evict(st):
    c = st["case"]
    page, budget = c["page"], c["budget"]
    kept = torch.full((c["batch"], c["hkv"], budget), -1, device="cuda", dtype=torch.int32)
    for b, n in enumerate(st["lens"]):
        keep = min(n, budget)
        w = st["weights"][b, :, :n]
        key = w.clone()
        key[:, :c["sink"]] = float("inf")
        key[:, max(0, n - c["recent"]):] = float("inf")
        best = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :keep]
        best = torch.sort(best, dim=1).values
        kept[b, :, :keep] = best
        st["weights_out"][b, :, :keep] = torch.gather(w, 1, best)
        st["weights_out"][b, :, keep:n] = 0
        to = torch.arange(keep, device="cuda")
        block, at = st["out_table"][b][to // page].long(), to % page
        for x in ("k_cache", "v_cache"):
            rows = torch.gather(_gather(st[x], st["table"][b], n), 1, best[..., None].expand(-1, -1, c["d"]))
            st[x][block, :, at] = rows.transpose(0, 1)
    return kept, st["seq_lens"].clamp(max=budget), st["weights_out"], st["k_cache"], st["v_cache"]


def _plain_logits(st):
    x = st["logits"].float()
    v = x.shape[1]
    at = torch.arange(st["history"].shape[1], device="cuda")
    valid = at < st["history_lens"][:, None]
    made = valid & (at >= st["prompt_lens"][:, None])
    ids = st["history"].long()
    seen = torch.zeros_like(x).scatter_add_(1, ids, valid.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, ids, made.float())
    r = st["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0)
    if st["bias"] is not None:
        x = x.scatter_add(1, st["bias_ids"].long(), st["bias"])
    if st["mask"] is not None:
        bits = (st["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = x.masked_fill(bits.flatten(1)[:, :v] == 0, float("-inf"))
    return x.to(st["logits"].dtype)


# ------------------------------------------------------------------- work --
def work(case):
    op = case["op"]
    size = _SIZE[case["dtype"]]
    if op == "append":
        n, heads = case["tokens"], case["hq"] + 2 * case["hkv"]
        return {"bytes": 2 * n * heads * case["d"] * size + 2 * 4 * case["half"] * n + n * (4 * case["axes"] + 8),
                "flops": 6 * n * (case["hq"] + case["hkv"]) * case["half"]}
    if op == "attend":
        lens = _lens(case)
        seen = sum(min(n, case["window"] or n) for n in lens)
        tables = sum(-(-min(n, case["window"] or n) // case["page"]) for n in lens)
        moved = 2 * seen * case["hkv"] * case["d"] * size + 2 * case["batch"] * case["hq"] * case["d"] * size
        moved += 4 * tables + 4 * case["batch"] + (4 * case["hq"] if case["alibi"] else 0)
        if case["weights"]:
            moved += 8 * sum(lens) * case["hkv"]
        return {"bytes": moved, "flops": 4 * seen * case["hq"] * case["d"]}
    if op == "evict":
        lens = _lens(case)
        keep = [min(n, case["budget"]) for n in lens]
        rows = 4 * sum(keep) * case["hkv"] * case["d"] * size
        pages = sum(-(-n // case["page"]) for n in lens + keep)
        return {"bytes": rows + case["hkv"] * (8 * sum(lens) + 4 * case["batch"] * case["budget"])
                + 4 * pages + 8 * case["batch"], "flops": sum(lens) * case["hkv"]}
    b, v = case["batch"], case["vocab"]
    lens, _ = _history_lens(case)
    return {"bytes": 2 * b * v * size + 4 * sum(lens) + 8 * b * case["bias"] + (4 * b * -(-v // 32) if case["mask"] else 0)
            + 20 * b, "flops": 4 * b * v}


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    """What ``run`` returns, from the definitions, in 64 bits."""
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict, "logits": _exact_logits}[case["op"]](st)


def _exact_append(st):
    page, n = st["case"]["page"], st["case"]["tokens"]
    half = st["cos"].shape[1]
    angle_cos = torch.empty((n, 1, half), device="cuda", dtype=torch.float64)
    angle_sin = torch.empty_like(angle_cos)
    at = 0
    for a, width in enumerate(st["sections"]):
        rows = st["positions"][a].long()
        angle_cos[:, 0, at:at + width] = st["cos"].index_select(0, rows)[:, at:at + width].double()
        angle_sin[:, 0, at:at + width] = st["sin"].index_select(0, rows)[:, at:at + width].double()
        at += width
    turn = torch.complex(angle_cos, angle_sin)

    def rotate(x):
        y = x.double().clone()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        return y

    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    flat_k, flat_v = (x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3]) for x in (kc, vc))
    flat_k.index_copy_(0, st["slots"], rotate(st["k"]))
    flat_v.index_copy_(0, st["slots"], st["v"].double())
    shape = (kc.shape[0], page, kc.shape[1], kc.shape[3])
    return rotate(st["q"]), flat_k.view(shape).transpose(1, 2), flat_v.view(shape).transpose(1, 2)


def _exact_attend(st):
    c = st["case"]
    hkv, d, page = c["hkv"], c["d"], c["page"]
    group = c["hq"] // hkv
    out = torch.empty((c["batch"], c["hq"], d), device="cuda", dtype=torch.float64)
    wout = st["weights_out"].double() if c["weights"] else None
    for b, n in enumerate(st["lens"]):
        t = torch.arange(n, device="cuda")
        if c["window"]:
            t = t[t > n - 1 - c["window"]]
        block, at = st["table"][b].long()[t // page], t % page
        if c["weights"]:
            wout[b, :, :n] = st["weights"][b, :, :n].double()
        for h in range(hkv):
            k, v = st["k_cache"][block, h, at].double(), st["v_cache"][block, h, at].double()
            rows = slice(h * group, (h + 1) * group)
            s = (k @ st["q"][b, rows].double().t()) / math.sqrt(d)
            if c["softcap"]:
                s = torch.tanh(s / c["softcap"]) * c["softcap"]
            if c["alibi"]:
                s = s - (n - 1 - t).double()[:, None] * st["slopes"][rows].double()
            p = torch.softmax(s, 0)
            out[b, rows] = p.t() @ v
            if c["weights"]:
                wout[b, h, t] += p.sum(1)
    return (out, wout) if c["weights"] else out


def _exact_evict(st):
    c = st["case"]
    page, budget = c["page"], c["budget"]
    kept = torch.full((c["batch"], c["hkv"], budget), -1, dtype=torch.int32)
    kc, vc, wout = st["k_cache"].double(), st["v_cache"].double(), st["weights_out"].double()
    weights = st["weights"].cpu().tolist()
    for b, n in enumerate(st["lens"]):
        keep = min(n, budget)
        for h in range(c["hkv"]):
            w = weights[b][h]
            last = max(0, n - c["recent"])
            must = [t for t in range(n) if t < c["sink"] or t >= last]
            rest = sorted((t for t in range(c["sink"], last)), key=lambda t: (-w[t], t))
            best = torch.tensor(sorted(must + rest[:max(0, keep - len(must))]))
            kept[b, h, :keep] = best
            src, dst = best.cuda(), torch.arange(keep, device="cuda")
            wout[b, h, :keep] = st["weights"][b, h, src].double()
            wout[b, h, keep:n] = 0
            sb, db = st["table"][b].long()[src // page], st["out_table"][b].long()[dst // page]
            kc[db, h, dst % page] = st["k_cache"][sb, h, src % page].double()
            vc[db, h, dst % page] = st["v_cache"][sb, h, src % page].double()
    lens = torch.tensor([min(n, budget) for n in st["lens"]], dtype=torch.int32)
    return kept.cuda(), lens.cuda(), wout, kc, vc


def _exact_logits(st):
    c = st["case"]
    x = st["logits"].double()
    v = c["vocab"]
    lens, prompt = _history_lens(c)
    for b in range(c["batch"]):
        ids = st["history"][b, :lens[b]].long()
        r, f, p = (st[k][b].double() for k in ("repetition", "frequency", "presence"))
        seen = torch.unique(ids)
        y = x[b, seen]
        x[b, seen] = torch.maximum(y, y.new_zeros(())) / r + torch.minimum(y, y.new_zeros(())) * r
        made, times = torch.unique(ids[prompt[b]:], return_counts=True)
        x[b, made] -= f * times + p
        if c["bias"]:
            x[b, st["bias_ids"][b].long()] += st["bias"][b].double()
        if c["mask"]:
            t = torch.arange(v, device="cuda")
            allowed = torch.bitwise_right_shift(st["mask"][b].long()[t // 32] & 0xFFFFFFFF, t % 32) % 2 == 1
            x[b, ~allowed] = float("-inf")
    return x
