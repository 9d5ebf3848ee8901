"""One decoding step over a paged cache, on the GPU, against 64-bit definitions.

Tolerances, in the order in which the terms arise (u = 2^-24, one fp32 rounding):

* A score is a sum of D products that are exact in fp32, rounded at most D
  times (twice u each where the tensor core truncates), then scaled, capped and
  biased with a handful of roundings. With A = max_t sum_d |scale q_d k_d| and S
  the largest score or bias, it is off by at most delta = 2u (D A + 8 S).
* exp of it is off by the factor e^delta, the exponential's own 2^-21 and the
  weight's 2^-16 (a 16-bit value and its 16-bit remainder, bf16 the coarser),
  numerator and denominator both: at most 2 delta + 2^-14 of sum p |v|.
* The result is rounded once to 16 bits: eps / 2 of it, 2^-25 where fp16 is subnormal.

Rotations round three times in fp32 and once to 16 bits; logits four times in
fp32 and once to their type; an eviction moves values and is exact.
"""
import math

import pytest
import torch

import oracle
from neso_b200 import _lib, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _make_cache(g, dtype, pages, hkv, page, D, layout="hnd"):
    """K and V with NaN everywhere; tests fill the visible tokens. Returns device tensors."""
    if layout == "hnd":
        k, v = (torch.full((pages, hkv, page, D), math.nan, dtype=dtype) for _ in range(2))
        return k.cuda(), v.cuda()
    if layout == "nhd":
        k, v = (torch.full((pages, page, hkv, D), math.nan, dtype=dtype).cuda().transpose(1, 2) for _ in range(2))
        return k, v
    both = torch.full((pages, 2, hkv, page, D + 8), math.nan, dtype=dtype).cuda()  # joint buffer, padded rows
    return both[:, 0, :, :, :D], both[:, 1, :, :, :D]


def _fill(g, cache, table, n, scale=1.0):
    """Random values for tokens 0..n-1 of one sequence."""
    page, hkv, D = cache.shape[2], cache.shape[1], cache.shape[3]
    x = (torch.randn(n, hkv, D, generator=g) * scale).to(cache.dtype).cuda()
    for t in range(0, n, page):
        m = min(page, n - t)
        cache[int(table[t // page]), :, :m] = x[t:t + m].transpose(0, 1)


def _setup(seed, dtype, lens, hq, hkv, D, page, layout="hnd", extra_width=0, spare=3):
    g = _gen(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    width = max(need + [0]) + extra_width
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)[:sum(need)].tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, m in enumerate(need):
        table[b, :m] = torch.tensor([order.pop() for _ in range(m)], dtype=torch.int32)
    k, v = _make_cache(g, dtype, pages, hkv, page, D, layout)
    for b, n in enumerate(lens):
        _fill(g, k, table[b], max(n, 0))
        _fill(g, v, table[b], max(n, 0))
    q = (torch.randn(len(lens), hq, D, generator=g) * 1.5).to(dtype).cuda()
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32), g


def _attention_tolerance(out, bounds, dtype, D, biggest):
    delta = 2 * U * (D * bounds[..., :1] + 8 * biggest)
    return (2 * delta + 2.0 ** -14) * bounds[..., 1:] + torch.finfo(dtype).eps / 2 * out.abs() + 2.0 ** -25


def _check_attention(q, k, v, table, lens, D, dtype, scale=None, softcap=0.0, window=0, slopes=None, weights=None,
                     **kw):
    s = 1 / math.sqrt(D) if scale is None else scale
    got = ops.paged_attention(q, k, v, table.cuda(), lens.cuda(), scale=scale, softcap=softcap, window=window,
                              slopes=None if slopes is None else slopes.cuda(), weights=weights, **kw)
    ref, sums, bounds = oracle.decode_attention(q.cpu(), k.cpu(), v.cpu(), table, lens, s, softcap, window, slopes)
    span = window if window else int(max(lens.max(), 0))
    biggest = float(bounds[..., 0].max()) + (float(slopes.abs().max()) * span if slopes is not None else 0.0)
    tol = _attention_tolerance(ref, bounds, dtype, D, biggest)
    err = (got.cpu().double() - ref).abs()
    assert got.dtype == dtype and bool((err <= tol).all()), float((err - tol).max())
    return got, sums, 2 * 2 * U * (D * float(bounds[..., 0].max()) + 8 * biggest) + 2.0 ** -19


# ------------------------------------------------------------ attention ----
ATTENTION = [
    # lens, hq, hkv, D, page
    ([1], 1, 1, 64, 16),
    ([1], 8, 1, 128, 16),
    ([0, 1, 2, 15, 16, 17, 33], 4, 2, 64, 16),
    ([129], 16, 16, 64, 16),
    ([700, 5, 0, 64, 1], 8, 1, 128, 7),
    ([40, 250], 9, 1, 64, 1),          # pages of one token, group of nine
    ([257, 31], 32, 2, 128, 24),       # group of sixteen, pages that end inside a unit
    ([100, 3], 20, 1, 64, 256),        # group of twenty: two passes of ten
    ([65, 300], 50, 1, 128, 32),       # group of fifty: four passes, the last short
    ([1000, 999, 998], 6, 2, 128, 128),
    ([0, 0], 4, 4, 64, 16),
    ([8000], 3, 1, 64, 64),            # clusters of sixteen CTAs per pair
    ([5000, 40], 32, 2, 128, 16),
    ([2000], 8, 2, 64, 16),            # clusters of eight, four and two CTAs per pair, and runs
    ([1500, 7, 0], 16, 4, 128, 16),
    ([300] * 9, 24, 8, 64, 24),
    ([9000], 4, 1, 128, 64),
    ([60] * 40, 12, 4, 64, 16),
    ([30, 70] * 40, 8, 4, 64, 16),     # more pairs than clusters take
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_attention_shapes(dev, case, dtype):
    lens, hq, hkv, D, page = ATTENTION[case]
    q, k, v, table, n, _ = _setup(case, dtype, lens, hq, hkv, D, page)
    _check_attention(q, k, v, table, n, D, dtype)


def test_attention_clusters_of_sixteen_are_found(dev):
    # very few pairs whose tables are too long for eight CTAs take sixteen, without a workspace,
    # where the device can hold such a cluster, and the workspace follows what the call then does
    need = _lib.lib().neso_paged_attention_workspace
    _lib.lib().neso_set_device(0)
    assert need(1, 3, 1, 64, 1000, 16, 0) == 0 and need(1, 16, 1, 128, 512, 16, 0) == 0
    assert need(1, 3, 1, 64, 1025, 16, 0) > 0 and need(8, 16, 1, 128, 1000, 16, 0) > 0
    assert _lib.last_error() == ""


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 15, 16, 17, 100])
def test_attention_window(dev, window, dtype):
    q, k, v, table, n, _ = _setup(window, dtype, [1, 16, 99, 100, 101, 333], 8, 2, 64, 24)
    # what the window hides may be anything
    for b, length in enumerate(n.tolist()):
        for t in range(max(0, length - window)):
            k[int(table[b, t // 24]), :, t % 24] = math.inf
            v[int(table[b, t // 24]), :, t % 24] = math.nan
    _check_attention(q, k, v, table, n, 64, dtype, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softcap,use_slopes,window", [(5.0, False, 0), (0.0, True, 0), (30.0, True, 50)])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_bias(dev, D, softcap, use_slopes, window, dtype):
    q, k, v, table, n, g = _setup(7, dtype, [200, 33, 1, 0], 12, 2, D, 16)
    slopes = torch.rand(12, generator=g) * 0.3 - 0.05 if use_slopes else None
    _check_attention(q, k, v, table, n, D, dtype, softcap=softcap, slopes=slopes, window=window)


@pytest.mark.parametrize("layout", ["nhd", "joint"])
def test_attention_strides(dev, layout):
    q, k, v, table, n, _ = _setup(11, torch.float16, [130, 17], 8, 4, 64, 16, layout=layout)
    wide = torch.full((2, 12, 72), math.nan, dtype=torch.float16, device=dev)  # q inside a fused projection
    wide[:, 2:10, :64] = q
    _check_attention(wide[:, 2:10, :64], k, v, table, n, 64, torch.float16)
    tw = torch.full((2, table.shape[1] + 5), 0, dtype=torch.int32, device=dev)
    tw[:, :table.shape[1]] = table.to(dev)
    a = ops.paged_attention(q, k, v, tw[:, :table.shape[1]], n.cuda())
    assert torch.equal(a, ops.paged_attention(q, k, v, table.cuda(), n.cuda()))


def test_attention_extreme_scores(dev):
    # one token far above the rest; scores of +-30000 at scale 1; -inf keys leave their token out
    q, k, v, table, n, _ = _setup(12, torch.float16, [90], 2, 2, 64, 16)
    q[:] = 0
    q[:, :, 0] = 60.0
    k[:, :, :, 0] = torch.where(k[:, :, :, 0].isnan(), k[:, :, :, 0], torch.full_like(k[:, :, :, 0], -500.0))
    t = 77
    k[int(table[0, t // 16]), :, t % 16, 0] = 500.0
    got = ops.paged_attention(q, k, v, table.cuda(), n.cuda(), scale=1.0)
    assert torch.equal(got[0], v[int(table[0, t // 16]), :, t % 16])
    k[int(table[0, 0]), :, 3, 0] = -math.inf
    assert torch.equal(got, ops.paged_attention(q, k, v, table.cuda(), n.cuda(), scale=1.0))
    # a NaN key that is visible shows
    k[int(table[0, 0]), 0, 3, 1] = math.nan
    got = ops.paged_attention(q, k, v, table.cuda(), n.cuda(), scale=1.0)
    assert bool(got[0, 0].isnan().all()) and not bool(got[0, 1].isnan().any())


def _uniform_pages(q, rows, values, dtype, dev):
    """A cache whose page i holds one key and one value in every row: the first
    element of the key is rows[i], every element of the value values[i]."""
    hkv, D = q.shape[1], q.shape[2]
    k = torch.zeros(len(rows), hkv, 16, D, dtype=dtype, device=dev)
    v = torch.zeros_like(k)
    for i, (x, y) in enumerate(zip(rows, values)):
        k[i, :, :, 0], v[i] = x, y
    return k, v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,hkv,D,n", [
    (64, 8, 128, 8192),   # runs of thousands of tokens
    (1, 3, 64, 8000),     # clusters
    (40, 4, 64, 900),     # a CTA per pair
])
def test_attention_sink_and_flat_tail(dev, B, hkv, D, n, dtype):
    # One token without a value 17.5 above the others (e^-17.5 = 2^-25.2): nearly
    # all of the weight is its own, and the result is what the others add up to.
    q = torch.zeros(B, 2 * hkv, D, dtype=dtype, device=dev)
    q[:, ::2, 0], q[:, 1::2, 0] = 1.0, 0.984375
    k, v = _uniform_pages(q[:, :hkv], [0.0, 0.0], [1.5, 1.5], dtype, dev)
    k[1, :, 5, 0], v[1, :, 5] = 17.5, 0.0  # page 1 has the sink
    table = torch.zeros(B, -(-n // 16), dtype=torch.int32, device=dev)
    table[:, table.shape[1] // 3] = 1
    got = ops.paged_attention(q, k, v, table, torch.full((B,), n, dtype=torch.int32, device=dev), scale=1.0)
    for row, top in ((slice(0, None, 2), 17.5), (slice(1, None, 2), 17.5 * 0.984375)):
        tail = (n - 1) * math.exp(-top)
        want = 1.5 * tail / (1 + tail)
        # sum p |v| is `want` itself; A = S = top, a sum of one product
        tol = (2 * 2 * U * (1 + 8) * top + 2.0 ** -14) * want + torch.finfo(dtype).eps / 2 * want + 2.0 ** -25
        assert float((got[:, row].double() - want).abs().max()) <= tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,page", [(64, 16), (128, 24)])
def test_attention_differences_of_close_weights(dev, D, page, dtype):
    # Values 1 and -1 of two tokens whose weights are nearly the same: the result
    # is the weights' difference, and shows how exactly they were held.
    B, hkv, n = 16, 4, 15
    q, k, v, table, lens, g = _setup(D, dtype, [n] * B, 2 * hkv, hkv, D, page)
    q[:] = 0
    q[:, ::2, 0], q[:, 1::2, 0], q[:, :, 1] = 1.0, 0.8125, 2.0 ** -12
    key, value = torch.zeros(B, hkv, n, D), torch.zeros(B, hkv, n, D)
    coarse, fine = -torch.rand(B, hkv, 7, generator=g), -torch.rand(B, hkv, 14, generator=g)
    key[:, :, 1::2, 0], key[:, :, 2::2, 0], key[:, :, 1:, 1] = coarse, coarse, fine
    pair = torch.arange(D) % 7
    value[:, :, 1 + 2 * pair, torch.arange(D)], value[:, :, 2 + 2 * pair, torch.arange(D)] = 1.0, -1.0
    rows = table[:, 0].long().to(dev)
    k[rows, :, :n], v[rows, :, :n] = key.to(dtype).to(dev), value.to(dtype).to(dev)
    got = ops.paged_attention(q, k, v, table.to(dev), lens.to(dev), scale=1.0).cpu().double()
    s = torch.einsum("bhgd,bhtd->bhgt", q.cpu().double().view(B, hkv, 2, D), key.to(dtype).double())
    p = torch.exp(s)  # the first token's score is 0, the others' lie in [-1 - 2^-12, 0]
    total = p.sum(-1, keepdim=True)
    a, b = p[..., 1 + 2 * pair], p[..., 2 + 2 * pair]
    want = ((a - b) / total).view(got.shape)
    # A score of two products: one sum (2 U), its scale and its product (2 U); the
    # exponential 2^-22 = 4 U; what the 16-bit parts leave, 4 U at most: 12 U of each
    # weight, and 4 U for the truncated sum of the two. The total's error is relative.
    tol = (28 * U * torch.maximum(a, b) / total).view(got.shape) + (torch.finfo(dtype).eps / 2 + 2.0 ** -16) * want.abs() + 2.0 ** -25
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,hkv", [(64, 16), (128, 8)])
def test_attention_long_sums(dev, D, hkv, dtype):
    # Values 1 and 1 + eps, equal weights (others for each query head): the result lies a
    # little above the middle between the two, so that a small loss on the way rounds it
    # down. As many equal segments as the grid has warps: each works through whole ones.
    units, B = 512, torch.cuda.get_device_properties(dev).multi_processor_count
    eps = torch.finfo(dtype).eps
    high = units // 2 + round(units * 4.6e-5 / eps)
    q = torch.zeros(B, 4 * hkv, D, dtype=dtype, device=dev)
    q[:, :, 0] = torch.linspace(0.5, 1.5, 4 * hkv)
    k, v = _uniform_pages(q[:, :hkv], [-0.625] * 3, [1.0, 1.0 + eps, 1.0], dtype, dev)
    k[2, :, 0, 0] = 0.0  # page 2 starts with the token that has the largest score
    table = torch.zeros(B, units, dtype=torch.int32, device=dev)
    table[:, torch.randperm(units - 1, generator=_gen(D))[:high].to(dev) + 1] = 1
    table[:, 0] = 2
    got = ops.paged_attention(q, k, v, table, torch.full((B,), 16 * units, dtype=torch.int32, device=dev), scale=1.0)
    c = torch.exp(-0.625 * q[0, :, 0].double())
    want = (1 + eps * 16 * high * c / (1 + (16 * units - 1) * c))[None, :, None]
    # Output and total take one rounding per unit, at most U of a sum that rises evenly: U / 2
    # of the whole per unit for each. Within a unit 16 products are cut off at 2 U of their
    # sum, 32 U; 16 U for the sums over lanes, the quotient and the parts of a join.
    tol = (units + 48) * U * want + eps / 2 * want
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())


def test_attention_bad_pages_and_lengths(dev):
    # pages outside the cache are left out, lengths are clamped to the table
    q, k, v, table, n, _ = _setup(13, torch.float16, [100, 64, 50, 40], 4, 2, 64, 16)
    table[0, 1], table[0, 5] = -7, 10 ** 6
    table[1, :] = -1
    n = torch.tensor([100, 64, -5, 2 ** 31 - 1], dtype=torch.int32)
    table[3, :] = table[3, 0]  # every page the same, so that all of the table is valid
    k[int(table[3, 0])] = 0.5
    v[int(table[3, 0])] = torch.randn(v.shape[1:], generator=_gen(1)).half().cuda()
    got, _, _ = _check_attention(q, k, v, table, n, 64, torch.float16)
    assert bool((got[1] == 0).all()) and bool((got[2] == 0).all())
    # no pages, no table: zeros
    empty = torch.empty(0, 2, 16, 64, dtype=torch.float16, device=dev)
    assert bool((ops.paged_attention(q, empty, empty, table.cuda(), n.cuda()) == 0).all())
    assert bool((ops.paged_attention(q, k, v, table[:, :0].cuda(), n.cuda()) == 0).all())
    assert ops.paged_attention(q[:0], k, v, table[:0].cuda(), n[:0].cuda()).shape == (0, 4, 64)


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("width", [3, 700])  # clusters, runs
def test_attention_empty_cache_and_q_off_16_bytes(dev, width, page):
    wide = torch.randn(2, 4, 66, generator=_gen(page)).half().to(dev)
    q = wide[:, :, 2:]
    empty = torch.empty(0, 2, page, 64, dtype=torch.float16, device=dev)
    table = torch.zeros(2, width, dtype=torch.int32, device=dev)
    n = torch.tensor([40, width * page], dtype=torch.int32, device=dev)
    assert bool((ops.paged_attention(q, empty, empty, table, n) == 0).all())
    w = torch.rand(2, 2, width * page, device=dev)
    before = w.clone()
    assert bool((ops.paged_attention(q, empty, empty, table, n, weights=w) == 0).all()) and torch.equal(w, before)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,D,window,extra", [(4, 4, 64, 0, 2), (8, 1, 128, 0, 2), (20, 1, 64, 0, 2), (6, 2, 128, 40, 2),
                                                   (8, 1, 128, 0, 700), (9, 1, 64, 40, 700), (16, 1, 64, 0, 200)])  # extra: a table for runs
def test_attention_weights(dev, hq, hkv, D, window, extra, dtype):
    lens = [0, 1, 31, 150, 700]
    q, k, v, table, n, g = _setup(hq, dtype, lens, hq, hkv, D, 16, extra_width=extra)
    tokens = table.shape[1] * 16 + 3
    before = torch.rand(5, hkv, tokens, generator=g)
    after = torch.full_like(before, -1.0).cuda()
    given = before.cuda()
    got, sums, tol = _check_attention(q, k, v, table, n, D, dtype, window=window, weights=given, weights_out=after)
    assert torch.equal(given.cpu(), before)
    plain = ops.paged_attention(q, k, v, table.cuda(), n.cuda(), window=window)
    assert torch.equal(plain, got)
    for b, length in enumerate(lens):
        for kv in range(hkv):
            add = torch.zeros(tokens, dtype=torch.float64)
            for t, x in sums.get((b, kv), {}).items():
                add[t] = x
            want = before[b, kv].double() + add
            bound = tol * add + 2 * U * want + 2.0 ** -60
            assert bool(((after[b, kv].cpu().double() - want).abs() <= bound)[:length].all())
            assert bool((after[b, kv, length:] == -1.0).all())
    ops.paged_attention(q, k, v, table.cuda(), n.cuda(), window=window, weights=given)
    for b, length in enumerate(lens):
        assert torch.equal(given[b, :, :length], after[b, :, :length])
        assert torch.equal(given[b, :, length:].cpu(), before[b, :, length:])


BIAS = [(5.0, False, 0), (0.0, True, 0), (30.0, True, 50), (0.0, True, 37), (8.0, False, 100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softcap,use_slopes,window", BIAS)
@pytest.mark.parametrize("D,hq,hkv,page", [(64, 12, 2, 16), (128, 8, 2, 24), (64, 24, 2, 8), (128, 12, 1, 16), (64, 20, 1, 16)])
def test_attention_bias_over_runs(dev, D, hq, hkv, page, softcap, use_slopes, window, dtype):
    # a table wide enough for runs, which pass from one ragged sequence to the next
    q, k, v, table, n, g = _setup(hq + D, dtype, [200, 33, 1, 0, 700, 17, 90], hq, hkv, D, page, extra_width=16000 // page)
    assert _lib.lib().neso_paged_attention_workspace(7, hq, hkv, D, table.shape[1], page, 0) > 0  # clusters need none
    slopes = torch.rand(hq, generator=g) * 0.3 - 0.05 if use_slopes else None
    _check_attention(q, k, v, table, n, D, dtype, softcap=softcap, slopes=slopes, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("softcap,use_slopes,window", BIAS)
@pytest.mark.parametrize("D,hq,hkv,extra", [(64, 12, 2, 2), (128, 12, 1, 2), (64, 12, 2, 1000), (128, 8, 2, 1000), (64, 24, 2, 1000),
                                            (128, 12, 1, 1000), (64, 20, 1, 1000)])  # 1000: a table for runs
def test_attention_weights_of_biased_scores(dev, D, hq, hkv, extra, softcap, use_slopes, window, dtype):
    lens = [0, 1, 31, 150, 700]
    q, k, v, table, n, g = _setup(hq + D, dtype, lens, hq, hkv, D, 16, extra_width=extra)
    slopes = torch.rand(hq, generator=g) * 0.3 - 0.05 if use_slopes else None
    before = torch.rand(5, hkv, table.shape[1] * 16, generator=g)
    after = torch.full_like(before, -1.0).cuda()
    _, sums, tol = _check_attention(q, k, v, table, n, D, dtype, softcap=softcap, slopes=slopes, window=window,
                                    weights=before.cuda(), weights_out=after)
    for b, length in enumerate(lens):
        for kv in range(hkv):
            add = torch.zeros(before.shape[2], dtype=torch.float64)
            for t, x in sums.get((b, kv), {}).items():
                add[t] = x
            want = before[b, kv].double() + add
            # The sum takes the query heads one after the other: a rounding of at most U of it for
            # each, hq / hkv in all, where a token's own share of the weight may be far smaller.
            bound = tol * add + (hq // hkv + 1) * U * want + 2.0 ** -60
            assert bool(((after[b, kv].cpu().double() - want).abs() <= bound)[:length].all())
            assert bool((after[b, kv, length:] == -1.0).all())


def test_attention_long_and_far(dev):
    # a cache of more than 2^32 elements, the sequences' pages at both ends; many runs per head are joined
    D, hkv, page, lens = 128, 8, 64, [20011, 37]
    pages = (1 << 32) // (2 * hkv * page * D) + 400
    both = torch.empty(pages, 2, hkv, page, D, dtype=torch.float16, device=dev)
    k, v = both[:, 0], both[:, 1]
    width = -(-lens[0] // page)
    table = torch.zeros(2, width, dtype=torch.int32)
    table[0] = torch.arange(pages - width, pages, dtype=torch.int32).flip(0)
    table[0, ::2] = torch.arange(0, width, dtype=torch.int32)[::2]
    table[1, 0] = pages - width - 1
    g = torch.Generator(device=dev).manual_seed(5)
    for b in range(2):
        rows = table[b, :-(-lens[b] // page)].long().to(dev)
        for c in (k, v):
            c[rows] = torch.randn(len(rows), hkv, page, D, device=dev, generator=g).half()
    q = torch.randn(2, 32, D, device=dev, generator=g).half()
    got = ops.paged_attention(q, k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev))
    for b in range(2):
        rows = table[b, :-(-lens[b] // page)].long().to(dev)
        kk, vv = (c[rows].transpose(0, 1).flatten(1, 2)[:, :lens[b]].double() for c in (k, v))
        qq = q[b].double().view(hkv, 4, D) / math.sqrt(D)
        p = torch.softmax(qq @ kk.transpose(1, 2), -1)
        ref = (p @ vv).view(32, D)
        big = float((qq.abs() @ kk.abs().transpose(1, 2)).max())
        bounds = torch.stack([torch.full((32,), big, dtype=torch.float64, device=dev),
                              (p @ vv.abs()).view(32, D).amax(-1)], -1)
        tol = _attention_tolerance(ref, bounds, torch.float16, D, big)
        assert bool(((got[b].double() - ref).abs() <= tol).all())


def test_attention_repeats_and_streams(dev):
    q, k, v, table, n, _ = _setup(21, torch.bfloat16, [500, 3, 900, 77] * 8, 16, 4, 128, 16)
    table, n = table.cuda(), n.cuda()
    first = ops.paged_attention(q, k, v, table, n)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(4):
        for s in streams:  # calls that overlap on the GPU have workspaces of their own
            with torch.cuda.stream(s):
                outs.append(ops.paged_attention(q, k, v, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_attention_graphs_follow_lengths(dev):
    q, k, v, table, n, _ = _setup(22, torch.float16, [300, 40], 8, 2, 64, 16)
    table, n = table.cuda(), n.cuda()
    w = torch.zeros(2, 2, table.shape[1] * 16, device=dev)
    ops.paged_attention(q, k, v, table, n)  # loads the kernels before the capture
    ops.paged_attention(q, k, v, table, n, weights=w.clone())
    graphs, outs = [], []
    pool_stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=pool_stream):
            outs.append(ops.paged_attention(q, k, v, table, n, weights=w))
        graphs.append(g)
    for lens in ([300, 40], [17, 0], [299, 1]):
        n.copy_(torch.tensor(lens, dtype=torch.int32))
        want_w = w.clone()
        want = ops.paged_attention(q, k, v, table, n, weights=want_w)
        ops.paged_attention(q, k, v, table, n, weights=want_w)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(w, want_w)


def test_attention_refusals(dev):
    q, k, v, table, n, _ = _setup(23, torch.float16, [20, 3], 4, 2, 64, 16)
    table, n = table.cuda(), n.cuda()
    call = ops.paged_attention
    with pytest.raises(TypeError):
        call(q.float(), k, v, table, n)
    with pytest.raises(TypeError):
        call(q, k, v, table.long(), n)
    with pytest.raises(TypeError):
        call(q, k, v.bfloat16(), table, n)
    with pytest.raises(ValueError):
        call(q.cpu(), k, v, table, n)
    with pytest.raises(ValueError):
        call(q, k, v, table, n.cpu())
    with pytest.raises(ValueError):
        call(q, k, v, table, n[:1])
    with pytest.raises(ValueError):
        call(q, k.transpose(2, 3), v.transpose(2, 3), table, n)
    with pytest.raises(ValueError):
        call(q, k, v, table, n, out=q)
    with pytest.raises(ValueError):
        call(q, k, v, table, n, weights=torch.zeros(2, 2, 31, device=dev))
    w = torch.zeros(2, 2, 100, device=dev)
    with pytest.raises(ValueError):
        call(q, k, v, table, n, weights=w[:, :, :64], weights_out=w[:, :, 1:65])
    with pytest.raises(_lib.NesoError, match="UNSUPPORTED"):
        call(q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), table, n)
    with pytest.raises(_lib.NesoError, match="multiple"):
        call(q[:, :3].contiguous(), k, v, table, n)
    with pytest.raises(_lib.NesoError, match="softcap"):
        call(q, k, v, table, n, softcap=-1.0)
    with pytest.raises(_lib.NesoError, match="window"):
        call(q, k, v, table, n, window=-1)
    odd = torch.zeros(k.numel() + 1, dtype=torch.float16, device=dev)[1:].view(k.shape)
    with pytest.raises(_lib.NesoError, match="MISALIGNED"):
        call(q, odd, v, table, n)


# --------------------------------------------------------------- append ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,hq,hkv,D,half,sections,page", [
    (1, 4, 2, 64, 32, None, 16),
    (7, 3, 1, 128, 64, [20, 22, 22], 5),
    (33, 2, 2, 64, 12, [12, 0], 16),       # a rotated part that is no multiple of eight
    (5, 1, 1, 80, 24, None, 1),
    (2, 1, 1, 64, 0, None, 16),            # nothing is rotated
    (300, 8, 8, 64, 32, None, 16),
    (1201, 1, 1, 16, 8, [3, 5], 16),       # tokens enough for several to a CTA, the last alone
])
def test_append(dev, N, hq, hkv, D, half, sections, page, dtype):
    g = _gen(N + D)
    q, k, v = ((torch.randn(N, h, D, generator=g) * 3).to(dtype) for h in (hq, hkv, hkv))
    axes = len(sections) if sections else 1
    angle = torch.rand(50, half, generator=g) * 6.28
    cos, sin = angle.cos(), angle.sin()
    pos = torch.randint(0, 50, (axes, N), generator=g, dtype=torch.int32)
    pages = -(-N // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:N]
    if N > 4:
        slots[2], slots[3] = -1, pages * page  # padding
        pos[0, 4] = 50                         # outside the table
    for fused in (False, True):
        if fused:
            buf = torch.cat([q, k, v], 1).cuda()
            qd, kd, vd = buf[:, :hq], buf[:, hq:hq + hkv], buf[:, hq + hkv:]
        else:
            qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
        kc, vc = (torch.full((pages, hkv, page, D), 7.0, dtype=dtype, device=dev) for _ in range(2))
        got = ops.rope_paged_append(qd, kd, vd, cos.cuda(), sin.cuda(), pos.cuda() if axes > 1 else pos[0].cuda(),
                                    slots.cuda(), kc, vc, sections=sections)
        refs = [oracle.decode_rope(x, cos, sin, pos, sections or [half]) for x in (q, k)]
        mags = [oracle.decode_rope(x.abs(), cos.abs(), -sin.abs(), pos, sections or [half]).abs() for x in (q, k)]
        want_k, want_v = (torch.full((pages, hkv, page, D), 7.0, dtype=torch.float64) for _ in range(2))
        tol_k = torch.zeros_like(want_k)
        eps = torch.finfo(dtype).eps / 2
        for i in range(N):
            s = int(slots[i])
            if 0 <= s < pages * page:
                want_k[s // page, :, s % page] = refs[1][i]
                # |u c| + |w s| bounds both rotated elements of a pair
                tol_k[s // page, :, s % page] = eps * refs[1][i].abs() + 6 * U * _pair_bound(mags[1][i], half) + 2.0 ** -25
                want_v[s // page, :, s % page] = v[i].double()
            else:
                refs[0][i] = 0
        tol_q = eps * refs[0].abs() + 6 * U * _pair_bound(mags[0], half) + 2.0 ** -25
        _close(got, refs[0], tol_q)
        _close(kc, want_k, tol_k)
        _close(vc, want_v, torch.zeros_like(want_v))


def _pair_bound(m, half):
    """The larger magnitude of each rotated pair, for both of its elements."""
    m = m.clone()
    top = torch.maximum(m[..., :half], m[..., half:2 * half])
    m[..., :half] = top
    m[..., half:2 * half] = top
    return m


def _close(got, want, tol):
    got = got.cpu().double()
    same_nan = torch.equal(got.isnan(), want.isnan())
    err = (got - want).abs()
    assert same_nan and bool((err <= tol)[~want.isnan()].all())


def test_append_in_place_streams_and_graph(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    q, k, v = (torch.randn(40, h, 64, device=dev, generator=g).half() for h in (4, 2, 2))
    cos, sin = torch.rand(64, 32, device=dev, generator=g), torch.rand(64, 32, device=dev, generator=g)
    pos = torch.arange(40, dtype=torch.int32, device=dev)
    slots = torch.arange(40, device=dev)
    kc, vc = (torch.zeros(4, 2, 16, 64, dtype=torch.float16, device=dev) for _ in range(2))
    want = ops.rope_paged_append(q, k, v, cos, sin, pos, slots, kc, vc)
    k1, v1 = kc.clone(), vc.clone()
    x = q.clone()
    assert ops.rope_paged_append(x, k, v, cos, sin, pos, slots, kc, vc, out=x) is x and torch.equal(x, want)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope_paged_append(q, k, v, cos, sin, pos, slots, kc, vc, out=out)
    kc.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(kc, k1) and torch.equal(vc, v1)
    # strided rows that are not on 16 bytes take the scalar form: same values
    wide = torch.empty(40, 8, 65, dtype=torch.float16, device=dev)
    wide[:, :4, 1:], wide[:, 4:6, 1:], wide[:, 6:, 1:] = q, k, v
    kc.zero_()
    got = ops.rope_paged_append(wide[:, :4, 1:], wide[:, 4:6, 1:], wide[:, 6:, 1:], cos, sin, pos, slots, kc, vc)
    assert torch.equal(got, want) and torch.equal(kc, k1)


def test_append_refusals(dev):
    q, k = torch.zeros(3, 4, 64, dtype=torch.float16, device=dev), torch.zeros(3, 2, 64, dtype=torch.float16, device=dev)
    cos = torch.zeros(10, 32, device=dev)
    pos, slots = torch.zeros(3, dtype=torch.int32, device=dev), torch.arange(3, device=dev)
    kc = torch.zeros(2, 2, 16, 64, dtype=torch.float16, device=dev)
    vc = kc.clone()
    call = ops.rope_paged_append
    with pytest.raises(TypeError):
        call(q, k, k, cos.double(), cos.double(), pos, slots, kc, vc)
    with pytest.raises(TypeError):
        call(q, k, k, cos, cos, pos, slots.int(), kc, vc)
    with pytest.raises(ValueError):
        call(q, k[:2], k, cos, cos, pos, slots, kc, vc)
    with pytest.raises(ValueError):
        call(q, k, k, cos, cos, torch.zeros(2, 3, dtype=torch.int32, device=dev), slots, kc, vc)
    with pytest.raises(ValueError):
        call(q, k, k, cos, cos, pos, slots, kc[:1].expand(2, 2, 16, 64), vc)
    big = torch.zeros(4, 4, 64, dtype=torch.float16, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        call(big[:3], k, k, cos, cos, pos, slots, kc, vc, out=big[1:])
    with pytest.raises(_lib.NesoError, match="sections"):
        call(q, k, k, cos, cos, torch.zeros(2, 3, dtype=torch.int32, device=dev), slots, kc, vc, sections=[16, 15])
    wide = torch.zeros(10, 40, device=dev)
    with pytest.raises(_lib.NesoError, match="rotates more"):
        call(q, k, k, wide, wide, pos, slots, kc, vc)


# ---------------------------------------------------------------- evict ----
def _check_evict(seed, dtype, lens, hkv, D, page, budget, recent, sink, mode, weights=None, layout="hnd", extra=0):
    q, k, v, table, n, g = _setup(seed, dtype, lens, hkv, hkv, D, page, layout=layout, extra_width=extra,
                                  spare=3 + len(lens) * (-(-budget // page)))
    tokens = table.shape[1] * page
    if weights is None:
        weights = torch.rand(len(lens), hkv, tokens, generator=g)
        weights = torch.where(weights < 0.2, torch.zeros(()), weights).mul(8).round().div(8)  # many ties
    before = weights.clone()
    kept_ref = oracle.decode_evict(before, n, budget, recent, sink, tokens)
    out_table = table
    if mode == "apart":
        free = sorted(set(range(k.shape[0])) - set(table[table >= 0].tolist()))
        width = -(-budget // page)
        out_table = torch.tensor(free[:len(lens) * width], dtype=torch.int32).view(len(lens), width)
    k0, v0 = k.cpu().clone(), v.cpu().clone()
    w = weights.cuda()
    w_out = torch.full_like(w, -3.0) if mode == "apart" else None
    kept, new = ops.kv_evict(k, v, table.cuda(), n.cuda(), w, budget, recent, sink=sink,
                             out_tables=out_table.cuda() if mode == "apart" else None, weights_out=w_out)
    after = w if w_out is None else w_out
    want_k, want_v = k0.clone(), v0.clone()
    want_w = before.clone() if w_out is None else torch.full_like(before, -3.0)
    for b, length in enumerate(lens):
        assert int(new[b]) == min(length, budget)
        for h in range(hkv):
            rows = kept_ref[b][h]
            assert kept[b, h].tolist() == rows + [-1] * (budget - len(rows))
            for j, t in enumerate(rows):
                src, dst = (int(table[b, t // page]), t % page), (int(out_table[b, j // page]), j % page)
                want_k[dst[0], h, dst[1]] = k0[src[0], h, src[1]]
                want_v[dst[0], h, dst[1]] = v0[src[0], h, src[1]]
            want_w[b, h, :len(rows)] = before[b, h, rows]
            want_w[b, h, len(rows):length] = 0
    torch.testing.assert_close(k.cpu(), want_k, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(v.cpu(), want_v, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(after.cpu(), want_w, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("mode", ["in_place", "apart"])
@pytest.mark.parametrize("lens,hkv,D,page,budget,recent,sink", [
    ([1], 1, 64, 16, 1, 0, 0),
    ([0, 1, 5, 17], 2, 64, 4, 5, 2, 1),
    ([100, 37, 64], 2, 128, 16, 32, 0, 0),
    ([100, 37, 64], 1, 128, 7, 32, 32, 0),     # nothing but the recent ones
    ([100, 37, 64], 1, 64, 7, 32, 10, 22),     # nothing is chosen
    ([333, 9], 3, 8, 24, 300, 100, 4),
    ([50], 1, 256, 16, 49, 0, 49),
    ([5000], 2, 64, 64, 4321, 17, 3),
    ([8192, 8193, 300], 1, 64, 64, 5000, 17, 3),  # on both sides of the change to counting together
    ([20000], 1, 8, 256, 12345, 1, 0),
])
def test_evict(dev, lens, hkv, D, page, budget, recent, sink, mode):
    _check_evict(len(lens) + D, TYPES[D % 3 % 2], lens, hkv, D, page, budget, recent, sink, mode)


@pytest.mark.parametrize("mode", ["in_place", "apart"])
def test_evict_special_weights(dev, mode):
    w = torch.zeros(2, 1, 64)
    w[0, 0] = torch.arange(64.0).flip(0) - 32.0
    w[0, 0, [5, 40]] = math.nan
    w[0, 0, [3, 60]] = math.inf
    w[0, 0, 7] = -math.inf
    w[1, 0, ::2] = -0.0  # ties with +0
    _check_evict(1, torch.float16, [64, 61], 1, 64, 16, 20, 3, 2, mode, weights=w)


def test_evict_strided_cache_and_spare_table(dev):
    _check_evict(2, torch.float16, [90, 20], 2, 64, 16, 30, 8, 2, "in_place", layout="nhd", extra=4)
    _check_evict(3, torch.float16, [90, 20], 2, 64, 16, 30, 8, 2, "apart", layout="joint", extra=4)


@pytest.mark.parametrize("keeps", ["all pages", "some pages"])
@pytest.mark.parametrize("lens,hkv,D,page,budget,recent,sink", [
    ([0, 1, 5, 17], 2, 64, 4, 5, 2, 1),
    ([333, 9], 3, 8, 24, 300, 100, 4),
    ([50, 90], 2, 256, 16, 49, 0, 40),
    ([300, 299], 2, 24, 1, 200, 3, 0),
    ([4096, 4000, 3000, 50], 8, 128, 16, 2048, 256, 4),
    ([9000], 1, 64, 64, 5000, 17, 3),
])
def test_evict_under_a_table_that_keeps_pages(dev, lens, hkv, D, page, budget, recent, sink, keeps):
    q, k, v, table, n, g = _setup(len(lens) + D, torch.float16, lens, hkv, hkv, D, page, spare=sum(-(-x // page) for x in lens))
    w = torch.rand(len(lens), hkv, table.shape[1] * page, generator=g).to(dev)
    width = -(-min(budget, table.shape[1] * page) // page)
    out = table[:, :width].clone()
    if keeps == "some pages":
        free = torch.tensor(sorted(set(range(k.shape[0])) - set(table[table >= 0].tolist())), dtype=torch.int32)
        fresh = (torch.rand(out.shape, generator=g) < 0.5) & (out >= 0)
        out[fresh] = free[:int(fresh.sum())]
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    table, n, out = table.to(dev), n.to(dev), out.to(dev)
    kept, new = ops.kv_evict(k, v, table, n, w, budget, recent, sink=sink, out_tables=out)
    for b in range(len(lens)):
        assert int(new[b]) == min(lens[b], budget)
        j = torch.arange(min(lens[b], budget), device=dev)
        for h in range(hkv):
            t = kept[b, h, :len(j)].long()
            for now, before in ((k, k0), (v, v0)):
                assert torch.equal(now[out[b, j // page].long(), h, j % page], before[table[b, t // page].long(), h, t % page])
            assert torch.equal(w[b, h, :len(j)], w0[b, h, t])
    if keeps == "all pages":  # the same as in place, wherever nothing was to be written too
        k1, v1, w1 = k0.clone(), v0.clone(), w0.clone()
        same, _ = ops.kv_evict(k1, v1, table, n, w1, budget, recent, sink=sink)
        assert torch.equal(same, kept) and torch.equal(w, w1)
        torch.testing.assert_close(k, k1, rtol=0, atol=0, equal_nan=True)
        torch.testing.assert_close(v, v1, rtol=0, atol=0, equal_nan=True)


def test_evict_bad_pages_and_lengths(dev):
    # rows on a page outside the cache are not moved; nothing else is touched
    q, k, v, table, n, g = _setup(4, torch.float16, [64], 1, 1, 64, 16)
    table[0, 2] = -1
    w = torch.zeros(1, 1, 64)
    w[0, 0, 40:44] = 1.0
    k0 = k.clone()
    kept, new = ops.kv_evict(k, v, table.cuda(), n.cuda(), w.cuda(), 10, 4)
    assert kept[0, 0].tolist() == [0, 1, 40, 41, 42, 43, 60, 61, 62, 63] and int(new[0]) == 10
    want = k0.clone()
    for j, t in enumerate(kept[0, 0].tolist()):
        if t // 16 != 2:
            want[int(table[0, 0]), 0, j] = k0[int(table[0, t // 16]), 0, t % 16]
    torch.testing.assert_close(k, want, rtol=0, atol=0, equal_nan=True)
    big = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=dev)
    table[0, 2] = 0
    _, new = ops.kv_evict(k, v, table.cuda(), big, w.cuda(), 64, 4)
    assert int(new[0]) == 64
    assert ops.kv_evict(k, v, table[:0].cuda(), n[:0].cuda(), w[:0].cuda(), 4, 0)[0].shape == (0, 1, 4)


def test_evict_refusals(dev):
    q, k, v, table, n, _ = _setup(5, torch.float16, [30], 2, 2, 64, 16)
    w = torch.zeros(1, 2, 32, device=dev)
    table, n = table.cuda(), n.cuda()
    for budget, recent, sink in ((0, 0, 0), (4, 5, 0), (4, 2, 3), (4, -1, 0)):
        with pytest.raises((_lib.NesoError, ValueError)):
            ops.kv_evict(k, v, table, n, w, budget, recent, sink=sink)
    with pytest.raises(ValueError):
        ops.kv_evict(k, v, table, n, w[:, :, :31], 8, 2)
    with pytest.raises(ValueError, match="out_tables"):
        ops.kv_evict(k, v, table, n, w, 20, 2, out_tables=table[:, :1])
    with pytest.raises(TypeError):
        ops.kv_evict(k, v, table, n, w.double(), 8, 2)
    wide = torch.zeros(1, 2, 40, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        ops.kv_evict(k, v, table, n, wide[:, :, :32], 8, 2, weights_out=wide[:, :, 4:36])


def test_evict_refuses_a_budget_beyond_its_steps(dev):
    q, k, v, table, n, _ = _setup(6, torch.float16, [30], 2, 2, 64, 16)
    w = torch.zeros(1, 2, 32, device=dev)
    with pytest.raises(ValueError, match="2\\^30"):  # refused before the 17 GB of `kept` are allocated
        ops.kv_evict(k, v, table.cuda(), n.cuda(), w, 2 ** 31 - 1, 2)


# --------------------------------------------------------------- logits ----
def _logit_inputs(seed, B, V, T, dtype, n_bias=5):
    g = _gen(seed)
    x = (torch.randn(B, V, generator=g) * 5).to(dtype)
    hist = torch.randint(0, max(1, min(V, 40)), (B, T), generator=g, dtype=torch.int32)
    hist[:, ::5] = torch.randint(0, V, hist[:, ::5].shape, generator=g, dtype=torch.int32)
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    lens[0] = T
    prompt = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    rep, freq, pres = 1 + torch.rand(B, generator=g), torch.rand(B, generator=g) - 0.3, torch.rand(B, generator=g)
    ids = torch.randint(0, V, (B, n_bias), generator=g, dtype=torch.int32)
    bias = torch.randn(B, n_bias, generator=g) * 3
    words = -(-V // 32)
    mask = torch.randint(-(1 << 31), 1 << 31, (B, words), generator=g).to(torch.int32)
    return x, dict(history=hist, history_lens=lens, prompt_lens=prompt, repetition=rep, frequency=freq, presence=pres,
                   bias_ids=ids, bias=bias, mask=mask)


def _check_logits(x, kw, xd=None, out=None):
    got = ops.process_logits(x.cuda() if xd is None else xd, out=out,
                             **{k: None if v is None else v.cuda() for k, v in kw.items()})
    want, mag = oracle.decode_logits(x, **kw)
    eps = torch.finfo(x.dtype).eps / 2
    n = kw["bias"].shape[1] if kw.get("bias") is not None else 0
    tol = (5 + n) * U * mag + eps * want.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    g = got.cpu().double()
    fin = want.isfinite()
    torch.testing.assert_close(g[~fin], want[~fin], rtol=0, atol=0, equal_nan=True)
    assert bool(((g - want).abs() <= tol)[fin].all())
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,V,T", [(1, 1, 1), (3, 31, 7), (2, 33, 50), (2, 8187, 100), (3, 8193, 64), (1, 20001, 300)])
def test_logits(dev, B, V, T, dtype):
    x, kw = _logit_inputs(V, B, V, T, dtype)
    kw["mask"][0] = 0 if B > 1 else -1  # a row whose mask leaves nothing
    _check_logits(x, kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,T,in_place", [(130, 16390, 200, False), (130, 16390, 200, True), (70, 33000, 17000, False),
                                            (70, 33000, 17000, True), (64, 32769, 9000, False)])
def test_logits_many_rows(dev, B, V, T, in_place, dtype):
    # rows enough for the long slices, histories of several rounds, other alignments and in place
    x, kw = _logit_inputs(V + T, B, V, T, dtype)
    kw["history"] = torch.randint(0, V, (B, T), generator=_gen(T), dtype=torch.int32)
    kw["mask"][::3], kw["mask"][1] = -1, 0
    rows = torch.tensor([0, 1, 2, B // 2, B - 1])  # rows are independent: a few are worked out in 64 bits
    wide = torch.zeros(B, V + 5, dtype=dtype, device=dev)
    wide[:, 3:3 + V] = x.cuda()
    xd = wide[:, 3:3 + V]
    d = {k: v.cuda() for k, v in kw.items()}
    got = ops.process_logits(xd, out=xd if in_place else None, **d)
    if in_place:
        assert bool((wide[:, :3] == 0).all()) and bool((wide[:, 3 + V:] == 0).all())
    want, mag = oracle.decode_logits(x[rows], **{k: v[rows] for k, v in kw.items()})
    g = got[rows.cuda()].cpu().double()
    fin = want.isfinite()
    torch.testing.assert_close(g[~fin], want[~fin], rtol=0, atol=0)
    tol = (5 + 5) * U * mag + torch.finfo(dtype).eps / 2 * want.abs()
    assert bool(((g - want).abs() <= tol)[fin].all())
    again = x.cuda()
    assert torch.equal(ops.process_logits(again, **d), got)  # other alignment, same values


def test_logits_many_rows_parts(dev):
    x, kw = _logit_inputs(77, 130, 16400, 60, torch.float32)
    rows = torch.tensor([0, 77, 129])
    for names in ((), ("mask",), ("bias_ids", "bias"), ("history", "history_lens", "prompt_lens", "presence", "repetition")):
        part = {k: v for k, v in kw.items() if k in names}
        want, mag = oracle.decode_logits(x[rows], **{k: v[rows] for k, v in part.items()})
        for xd in (x.cuda(), x.cuda()):
            got = ops.process_logits(xd, out=xd if names else None, **{k: v.cuda() for k, v in part.items()})
            g = got[rows.cuda()].cpu().double()
            fin = want.isfinite()
            assert torch.equal(g[~fin], want[~fin]) and bool(((g - want).abs() <= 11 * U * mag)[fin].all())


@pytest.mark.parametrize("names", [(), ("mask",), ("bias_ids", "bias"), ("history", "history_lens", "repetition"),
                                   ("history", "history_lens", "frequency"),
                                   ("history", "history_lens", "prompt_lens", "presence")])
def test_logits_parts(dev, names):
    x, kw = _logit_inputs(5, 2, 700, 90, torch.float32)
    _check_logits(x, {k: v for k, v in kw.items() if k in names})


def test_logits_odd_indexes(dev):
    # ids outside the vocabulary are skipped, lengths clamped, the same biased token adds up in order
    x, kw = _logit_inputs(6, 3, 500, 40, torch.float32)
    kw["history"][:, 3], kw["history"][:, 4], kw["history"][:, 5] = -1, 500, 2 ** 31 - 1
    kw["history_lens"] = torch.tensor([-4, 1000, 40], dtype=torch.int32)
    kw["prompt_lens"] = torch.tensor([0, -3, 1000], dtype=torch.int32)
    kw["bias_ids"] = torch.tensor([[7, 7, -1, 7, 499]] * 3, dtype=torch.int32)
    kw["mask"][:, 0] |= 128
    _check_logits(x, kw)
    x[0, 0], x[0, 1], x[0, 2] = math.inf, -math.inf, math.nan
    kw["mask"] = torch.full((3, 16), -1, dtype=torch.int32)
    got = _check_logits(x, kw)
    assert bool(got[0, 2].isnan())
    kw["mask"] = torch.zeros(3, 20, dtype=torch.int32)
    assert bool((_check_logits(x, kw) == -math.inf).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_strides_and_in_place(dev, dtype):
    x, kw = _logit_inputs(8, 4, 9001, 30, dtype)
    base = _check_logits(x, kw)
    for shift in (1, 3):  # rows off the vector boundary, odd pitch
        wide = torch.zeros(4, 9011, dtype=dtype, device=dev)
        view = wide[:, shift:shift + 9001]
        view.copy_(x)
        assert torch.equal(_check_logits(x, kw, xd=view), base)
        other = torch.zeros(4, 9011, dtype=dtype, device=dev)
        assert torch.equal(_check_logits(x, kw, xd=view, out=other[:, shift:shift + 9001]), base)
        assert bool((other[:, :shift] == 0).all()) and bool((other[:, shift + 9001:] == 0).all())
        assert torch.equal(_check_logits(x, kw, xd=view, out=view), base)
        assert bool((wide[:, :shift] == 0).all()) and bool((wide[:, shift + 9001:] == 0).all())


def test_in_place_views_of_one_row_whose_batch_strides_differ(dev):
    # the stride of a dimension of one has no meaning: these are the same tensor
    x, kw = _logit_inputs(10, 1, 100, 20, torch.float32)
    buf = torch.zeros(1, 128, device=dev)
    view = buf[:, :100]
    view.copy_(x)
    same = view.as_strided((1, 100), (100, 1))
    assert view.stride() != same.stride()
    want = ops.process_logits(x.cuda(), **{k: t.cuda() for k, t in kw.items()})
    assert _check_logits(x, kw, xd=view, out=same) is same and torch.equal(view, want)
    q, k, v, table, n, g = _setup(24, torch.float16, [20], 4, 2, 64, 16)
    w = torch.rand(2, 2, 50, generator=g).cuda()
    one = w[:1, :, :32]
    other = one.as_strided((1, 2, 32), (1, 50, 1))
    before = one.clone()
    ops.paged_attention(q, k, v, table.cuda(), n.cuda(), weights=one, weights_out=other)
    ops.paged_attention(q, k, v, table.cuda(), n.cuda(), weights=before)
    assert torch.equal(one, before)


def test_logits_graph(dev):
    x, kw = _logit_inputs(9, 2, 4000, 50, torch.float32)
    kw = {k: v.cuda() for k, v in kw.items()}
    x = x.cuda()
    want = ops.process_logits(x, **kw)
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.process_logits(x, out=out, **kw)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    kw["history_lens"].fill_(3)
    g.replay()
    assert torch.equal(out, ops.process_logits(x, **kw))


def test_logits_refusals(dev):
    x = torch.zeros(2, 100, device=dev)
    ids = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        ops.process_logits(x.double())
    with pytest.raises(ValueError):
        ops.process_logits(x, history=ids)
    with pytest.raises(ValueError):
        ops.process_logits(x, repetition=torch.ones(2, device=dev))
    with pytest.raises(ValueError):
        ops.process_logits(x, bias_ids=ids)
    with pytest.raises(ValueError):
        ops.process_logits(x, mask=torch.zeros(2, 3, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        ops.process_logits(x.t())
    with pytest.raises(ValueError, match="overlap"):
        big = torch.zeros(2, 128, device=dev)
        ops.process_logits(big[:, :100], out=big[:, 1:101])


def test_outputs_that_touch_other_inputs_are_refused(dev):
    q, k, v, table, n, g = _setup(25, torch.float16, [20, 3], 8, 2, 64, 16)
    table, n = table.to(dev), n.to(dev)
    slopes = torch.zeros(8, device=dev)
    w = torch.zeros(2, 2, 40, device=dev)
    page = k.flatten()[:1024].view(2, 8, 64)  # the output's shape, over the cache
    far = v.flatten()[-1024:].view(2, 8, 64)
    attend = ops.paged_attention
    for out in (page, far):
        with pytest.raises(ValueError, match="out overlaps [kv]_cache"):
            attend(q, k, v, table, n, out=out)
    big = torch.zeros(4096, device=dev)  # 32-bit words seen as other things
    half = big.view(torch.float16)[:1024].view(2, 8, 64)
    for name, kw in (("slopes", dict(slopes=big[500:508])), ("weights", dict(weights=big[100:260].view(2, 2, 40), weights_out=w))):
        with pytest.raises(ValueError, match=f"out overlaps {name}"):
            attend(q, k, v, table, n, out=half, **kw)
    with pytest.raises(ValueError, match="out overlaps block_tables"):
        attend(q, k, v, big.view(torch.int32)[:4].view(2, 2), n, out=half)
    with pytest.raises(ValueError, match="weights_out overlaps q"):
        attend(half, k, v, table, n, weights=w, weights_out=big[300:460].view(2, 2, 40))
    with pytest.raises(ValueError, match="weights_out overlaps k_cache"):
        kb = big.view(torch.float16)[:8192].view(4, 2, 16, 64)
        attend(q, kb, kb.clone(), table, n, weights=w, weights_out=big[300:460].view(2, 2, 40))
    with pytest.raises(ValueError, match="weights_out overlaps v_cache"):
        ops.kv_evict(kb.clone(), kb, table, n, w, 8, 2, weights_out=big[300:460].view(2, 2, 40))
    with pytest.raises(ValueError, match="overlap itself"):
        ops.kv_evict(k, v, table, n, w, 8, 2, weights_out=torch.zeros(200, device=dev).as_strided((2, 2, 40), (40, 20, 1)))
    with pytest.raises(ValueError, match="overlap itself"):
        ops.kv_evict(k.as_strided(k.shape, (1024, 512, 64, 1)), v, table, n, w, 8, 2)
    cos, pos, slots = torch.zeros(10, 32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), torch.arange(2, device=dev)
    new = torch.zeros(2, 8 * 64 + 2 * 2 * 64, dtype=torch.float16, device=dev)
    nk, nv = new[:, 512:640].view(2, 2, 64), new[:, 640:].view(2, 2, 64)
    append = ops.rope_paged_append
    for out, name in ((page, "k_cache"), (far, "v_cache"), (new.flatten()[:1024].view(2, 8, 64), "k")):
        with pytest.raises(ValueError, match=f"out overlaps {name}"):
            append(q, nk, nv, cos, cos, pos, slots, k, v, out=out)
    with pytest.raises(ValueError, match="out overlaps sin"):
        append(q, nk, nv, cos, big[:320].view(10, 32), pos, slots, k, v, out=half)
    x = torch.zeros(2, 100, device=dev)
    out = big[:200].view(2, 100)
    ids = big.view(torch.int32)[:6].view(2, 3)
    some = torch.zeros(2, dtype=torch.int32, device=dev)
    for name, kw in (("history", dict(history=ids, history_lens=some)), ("mask", dict(mask=big.view(torch.int32)[:8].view(2, 4))),
                     ("bias", dict(bias_ids=ids.clone(), bias=big[190:196].view(2, 3))),
                     ("presence", dict(history=ids.clone(), history_lens=some, presence=big[199:201]))):
        with pytest.raises(ValueError, match=f"out overlaps {name}"):
            ops.process_logits(x, out=out, **kw)
    with pytest.raises(ValueError, match="overlap itself"):
        ops.process_logits(x, out=big[:200].as_strided((2, 100), (60, 1)))


def test_outputs_between_the_pages_of_a_buffer(dev):
    # pages and other things in one buffer: an output in the room that the pages leave is apart from them
    q, k, v, table, n, g = _setup(26, torch.float16, [40, 3], 8, 2, 64, 16)
    buf = torch.zeros(k.shape[0], 2 * 2048 + 1024 + 256, dtype=torch.float16, device=dev)
    kb, vb = (buf[:, i * 2048:(i + 1) * 2048].view(-1, 2, 16, 64) for i in range(2))
    kb.copy_(k), vb.copy_(v)
    out = buf[1, 4096:5120].view(2, 8, 64)
    w = buf.view(torch.float32)[2, 2560:2688].view(2, 2, 32)
    w2 = torch.zeros(2, 2, 48, device=dev)
    table, n = table.to(dev), n.to(dev)
    assert ops.paged_attention(q, kb, vb, table, n, weights=w2, out=out) is out
    assert torch.equal(out, ops.paged_attention(q, k, v, table, n))
    short = torch.tensor([16, 3], dtype=torch.int32, device=dev)
    w.zero_()
    ops.kv_evict(kb, vb, table[:, :2], short, w2[:, :, :32], 4, 2, weights_out=w)
    assert torch.equal(out, ops.paged_attention(q, k, v, table, n)) and float(w[0].abs().sum()) > 0
    # heads that share one key: a view with a stride of 0 is read, beside a given output
    one, val = k[:, :1].expand(-1, 2, -1, -1), v[:, :1].expand(-1, 2, -1, -1)
    given = torch.empty_like(q)
    ops.paged_attention(q, one, val, table, n, out=given)
    assert torch.equal(given, ops.paged_attention(q, one.contiguous(), val.contiguous(), table, n))


# ------------------------------------------------------ torch operators ----
def test_torch_operators_match_tensor_api(dev):
    import neso_b200.torch_ops  # noqa: F401
    neso = torch.ops.neso
    q, k, v, table, n, g = _setup(31, torch.float16, [90, 20], 4, 2, 64, 16)
    table, n = table.cuda(), n.cuda()
    w = torch.rand(2, 2, table.shape[1] * 16, generator=g).cuda()
    w1, w2 = w.clone(), w.clone()
    a = neso.paged_attention(q, k, v, table, n, 0.125, 20.0, 30, None, w1)
    assert torch.equal(a, ops.paged_attention(q, k, v, table, n, 0.125, softcap=20.0, window=30, weights=w2))
    assert torch.equal(w1, w2) and not torch.equal(w1, w)
    b = neso.paged_attention(q, k, v, table, n, 0.125, 0.0, 0, torch.zeros(4, device=dev), None)
    assert b.shape == q.shape
    x, kw = _logit_inputs(32, 2, 500, 40, torch.float16)
    kw = {name: t.cuda() for name, t in kw.items()}
    assert torch.equal(neso.process_logits(x.cuda(), *kw.values()), ops.process_logits(x.cuda(), **kw))
    k1, v1, k2, v2 = k.clone(), v.clone(), k.clone(), v.clone()
    new = torch.randn(2, 8, 64, generator=g).half().cuda()
    ang = torch.rand(50, 32, generator=g).cuda()
    pos, slots = torch.tensor([3, 4], dtype=torch.int32, device=dev), torch.tensor([5, 20], device=dev)
    args = (new[:, :4], new[:, 4:6], new[:, 6:], ang, ang, pos, slots)
    assert torch.equal(neso.rope_paged_append(*args, k1, v1, None), ops.rope_paged_append(*args, k2, v2))
    torch.testing.assert_close(k1, k2, rtol=0, atol=0, equal_nan=True)
    r1 = neso.kv_evict(k1, v1, table, n, w1, 24, 4, 2, None)
    r2 = ops.kv_evict(k2, v2, table, n, w2, 24, 4, sink=2)
    assert torch.equal(r1[0], r2[0]) and torch.equal(r1[1], r2[1]) and torch.equal(w1, w2)
    torch.testing.assert_close(v1, v2, rtol=0, atol=0, equal_nan=True)
    for op, args in ((neso.paged_attention.default, (q, k1, v1, table, n, 0.1, 0.0, 0, None, w1)),
                     (neso.kv_evict.default, (k1, v1, table, n, w1, 24, 4, 2, None)),
                     (neso.process_logits.default, (x.cuda(), *kw.values()))):
        torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


# ------------------------------------------------------------- together ----
def test_decoding_steps_together(dev):
    """Prompt, a few decoding steps, an eviction, more steps: the cache, the
    accumulated weights and the outputs follow the 64-bit definitions."""
    D, hq, hkv, page, B, V = 64, 4, 2, 16, 2, 300
    g = _gen(99)
    lens = [37, 20]
    tables = torch.arange(8, dtype=torch.int32).view(2, 4).flip(0).contiguous()
    kc, vc = (torch.zeros(8, hkv, page, D, dtype=torch.float16, device=dev) for _ in range(2))
    angle = torch.rand(200, 32, generator=g) * 6.28
    cos, sin = angle.cos(), angle.sin()
    weights = torch.zeros(B, hkv, 64, device=dev)
    n = torch.zeros(B, dtype=torch.int32, device=dev)
    history = torch.zeros(B, 80, dtype=torch.int32)

    def append(counts, positions):
        N = sum(counts)
        q, k, v = (torch.randn(N, h, D, generator=g).half() for h in (hq, hkv, hkv))
        slots, i = torch.empty(N, dtype=torch.int64), 0
        for b, c in enumerate(counts):
            for t in range(int(n[b]), int(n[b]) + c):
                slots[i] = int(tables[b, t // page]) * page + t % page
                i += 1
        pos = torch.tensor(positions, dtype=torch.int32)
        out = ops.rope_paged_append(q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(), pos.cuda(), slots.cuda(), kc, vc)
        n.add_(torch.tensor(counts, dtype=torch.int32, device=dev))
        return out

    append(lens, [t for c in lens for t in range(c)])
    at = list(lens)
    for step in range(8):
        q = append([1, 1], at)
        at = [a + 1 for a in at]
        before = weights.cpu().double()
        out, sums, tol = _check_attention(q, kc, vc, tables, n.cpu(), D, torch.float16, weights=weights)
        for (b, kv), row in sums.items():
            for t, x in row.items():
                want = float(before[b, kv, t]) + x
                assert abs(float(weights[b, kv, t]) - want) <= tol * x + 2 * U * want
        logits = (torch.randn(B, V, generator=g) * 3)
        history[:, step] = torch.randint(0, V, (B,), generator=g, dtype=torch.int32)
        _check_logits(logits, dict(history=history, history_lens=torch.full((B,), step + 1, dtype=torch.int32),
                                   repetition=torch.full((B,), 1.2), presence=torch.full((B,), 0.5)))
        if step == 3:
            kept_ref = oracle.decode_evict(weights.cpu(), n.cpu(), 24, 6, 2, 64)
            w0 = weights.cpu().clone()
            kept, new = ops.kv_evict(kc, vc, tables.cuda(), n, weights, 24, 6, sink=2)
            for b in range(B):
                for h in range(hkv):
                    rows = kept_ref[b][h]
                    assert kept[b, h, :len(rows)].tolist() == rows
                    assert torch.equal(weights[b, h, :len(rows)].cpu(), w0[b, h, rows])
            n = new
            assert n.tolist() == [24, 24]
            assert bool((weights[:, :, 24:41] == 0).all())
