"""The decoding-step operators without a GPU: the C entry points refuse bad
calls before they touch a device, the tensor API refuses what is not a CUDA
tensor, the operators trace with fake tensors, and the 64-bit definitions that
the GPU tests compare with agree with hand-worked cases."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import neso_b200.torch_ops  # noqa: F401
import oracle
from neso_b200 import _lib, ops

I, U, M = _lib.NESO_ERR_INVALID_ARG, _lib.NESO_ERR_UNSUPPORTED, _lib.NESO_ERR_MISALIGNED
P = 1 << 20  # stands for a device pointer: every call below is refused or empty before one is used


def _attention(**kw):
    a = dict(q=P, k=P, v=P, tables=P, lens=P, slopes=None, win=None, wout=None, out=P, ws=P, ws_bytes=1 << 40, dtype=0,
             B=2, Hq=8, Hkv=2, D=64, scale=0.125, softcap=0.0, window=0, q_sb=512, q_sh=64, pages=4, page=16, ks=(2048, 1024, 64),
             vs=(2048, 1024, 64), width=3, ts=3, w=(0, 0, 0, 0))
    a.update(kw)
    return _lib.lib().neso_paged_attention(
        a["q"], a["k"], a["v"], a["tables"], a["lens"], a["slopes"], a["win"], a["wout"], a["out"], a["ws"], a["ws_bytes"],
        a["dtype"], a["B"], a["Hq"], a["Hkv"], a["D"], a["scale"], a["softcap"], a["window"], a["q_sb"], a["q_sh"],
        a["pages"], a["page"], *a["ks"], *a["vs"], a["width"], a["ts"], *a["w"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), I), (dict(Hq=7), I), (dict(Hkv=0), I), (dict(D=96), U), (dict(page=0), I), (dict(B=-1), I),
    (dict(window=-1), I), (dict(softcap=-0.5), I), (dict(softcap=math.nan), I), (dict(softcap=math.inf), I), (dict(softcap=1e-38), I),
    (dict(win=P), I), (dict(wout=P), I), (dict(q=None), I), (dict(lens=None), I), (dict(out=None), I),
    (dict(tables=None), I), (dict(k=None), I), (dict(k=P + 8), M), (dict(ks=(2048, 1024, 60)), M), (dict(vs=(2044, 1024, 64)), M),
    (dict(ks=(-2048, 1024, 64)), I), (dict(q=P + 2), M), (dict(q_sh=63), M), (dict(out=P + 2), M), (dict(ws=None, width=4000), I),
    (dict(ws_bytes=16, width=4000), I), (dict(ws=P + 4), M), (dict(pages=-1), I),
    (dict(B=1 << 16, Hq=1 << 10, Hkv=1 << 10, width=1 << 20), U),
    (dict(B=0), _lib.NESO_OK),
])
def test_attention_entry_refuses_before_the_device(kw, code):
    assert _attention(**kw) == code
    assert (code == _lib.NESO_OK) == (_lib.last_error() == "")


def test_attention_workspace():
    f = _lib.lib().neso_paged_attention_workspace
    assert f(2, 8, 3, 64, 4, 16, 0) == I and f(2, 8, 2, 96, 4, 16, 0) == U
    assert 0 == f(2, 8, 2, 64, 4, 16, 0) < f(2, 8, 2, 64, 4, 16, 1)  # short tables: clusters join by themselves
    assert 0 < f(2, 8, 2, 64, 4000, 16, 0) < f(2, 8, 2, 64, 4000, 16, 1)
    # scores of every query head and token of the table
    assert f(3, 8, 2, 64, 100, 16, 1) - f(3, 8, 2, 64, 100, 16, 0) >= 3 * 8 * 1600 * 4


def _append(**kw):
    a = dict(p=[P] * 10, dtype=0, N=3, Hq=4, Hkv=2, D=64, half=32, rows=10, axes=1, sections=None, st=(256, 64, 128, 64, 128, 64),
             pages=4, page=16, kc=(2048, 1024, 64), vc=(2048, 1024, 64))
    a.update(kw)
    return _lib.lib().neso_rope_paged_append(*a["p"], a["dtype"], a["N"], a["Hq"], a["Hkv"], a["D"], a["half"], a["rows"],
                                             a["axes"], a["sections"], *a["st"], a["pages"], a["page"], *a["kc"], *a["vc"], None)


def _ints(*x):
    return (_lib.ctypes.c_int32 * len(x))(*x)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), I), (dict(N=-1), I), (dict(D=60), U), (dict(D=2048), U), (dict(half=33), I), (dict(page=0), I),
    (dict(axes=0), I), (dict(axes=5), I), (dict(axes=2), I), (dict(axes=2, sections=_ints(16, 15)), I),
    (dict(axes=2, sections=_ints(33, -1)), I), (dict(sections=_ints(31)), I), (dict(p=[None] + [P] * 9), I),
    (dict(p=[P] * 6 + [None] + [P] * 3), I), (dict(p=[P] * 8 + [P + 2, P]), M), (dict(kc=(2048, 1024, 4)), M),
    (dict(Hq=70000), U), (dict(N=0), _lib.NESO_OK),
])
def test_append_entry_refuses_before_the_device(kw, code):
    assert _append(**kw) == code


def _evict(**kw):
    a = dict(p=[P] * 9, B=2, Hkv=2, D=64, budget=8, recent=2, sink=1, pages=4, page=16, ks=(2048, 1024, 64), vs=(2048, 1024, 64),
             width=3, ts=3, ow=3, os=3, w=(96, 48, 96, 48))
    a.update(kw)
    return _lib.lib().neso_kv_evict(*a["p"], a["B"], a["Hkv"], a["D"], a["budget"], a["recent"], a["sink"], a["pages"],
                                    a["page"], *a["ks"], *a["vs"], a["width"], a["ts"], a["ow"], a["os"], *a["w"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(budget=0), I), (dict(recent=8), I), (dict(sink=-1), I), (dict(recent=-1), I), (dict(recent=2 ** 31 - 1, sink=2 ** 31 - 1), I),
    (dict(D=60), U), (dict(D=264), U), (dict(page=0), I), (dict(Hkv=0), I), (dict(p=[P] * 4 + [None] + [P] * 4), I),
    (dict(p=[P] * 5 + [None] + [P] * 3), I), (dict(p=[P + 4] + [P] * 8), M), (dict(B=1 << 30), U), (dict(B=0), _lib.NESO_OK),
])
def test_evict_entry_refuses_before_the_device(kw, code):
    assert _evict(**kw) == code


def test_evict_entry_refuses_budgets_that_steps_of_a_row_would_pass_32_bits_with():
    assert _evict(budget=2 ** 31 - 1) == U and _evict(budget=2 ** 30 + 1) == U
    assert "2^30" in _lib.last_error()
    assert _evict(budget=2 ** 30, B=0) == _lib.NESO_OK


def test_evict_entry_refuses_weights_that_end_before_the_table():
    # three pages of 16 tokens: rows of 40 weights, in the batch or per kv head
    assert _evict(w=(96, 40, 96, 48)) == I and "48 tokens" in _lib.last_error()
    assert _evict(w=(40, 0, 96, 48)) == I
    assert _evict(w=(80, 0, 96, 48), Hkv=1, B=0) == _evict(w=(0, 0, 96, 48), B=0) == _lib.NESO_OK


def test_logits_entry_refuses_before_the_device():
    def f(x=P, out=P, dtype=2, B=2, V=100, hist=None, lens=None, T=0, ids=None, bias=None, n=0):
        return _lib.lib().neso_process_logits(x, out, dtype, B, V, V, V, hist, lens, None, T, T, None, None, None, ids, bias,
                                              n, None, 0, None)
    assert f(dtype=3) == I and f(B=-1) == I and f(hist=P, T=4) == I and f(ids=P, n=2) == I and f(bias=P, n=2) == I
    assert f(x=None) == I and f(out=None) == I and f(T=1 << 30, hist=P, lens=P) == U
    assert f(B=1 << 30, V=1 << 20) == U
    assert f(B=0) == _lib.NESO_OK and f(V=0) == _lib.NESO_OK


def test_tensor_api_refuses_what_is_not_on_a_gpu():
    x = torch.zeros(2, 4, 64, dtype=torch.float16)
    c = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    t, n = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    calls = [lambda: ops.paged_attention(x, c, c, t, n), lambda: ops.kv_evict(c, c, t, n, torch.zeros(2, 2, 16), 4, 1),
             lambda: ops.process_logits(torch.zeros(2, 8)),
             lambda: ops.rope_paged_append(x, x[:, :2], x[:, :2], torch.zeros(4, 32), torch.zeros(4, 32), n, n.long(), c, c)]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        ops.process_logits([1.0])
    with pytest.raises(TypeError):
        ops.paged_attention(None, c, c, t, n)


def test_fake_shapes_and_dtypes():
    with FakeTensorMode():
        def e(*shape, dtype=torch.float16):
            return torch.empty(shape, dtype=dtype, device="cuda")
        q, k, c = e(5, 8, 128), e(5, 2, 128), e(9, 2, 16, 128)
        ang, pos, slots = e(40, 64, dtype=torch.float32), e(3, 5, dtype=torch.int32), e(5, dtype=torch.int64)
        o = torch.ops.neso.rope_paged_append(q, k, k, ang, ang, pos, slots, c, c.clone(), [20, 22, 22])
        assert o.shape == q.shape and o.dtype == torch.float16
        t, n, w = e(5, 7, dtype=torch.int32), e(5, dtype=torch.int32), e(5, 2, 112, dtype=torch.float32)
        for weights in (None, w):
            o = torch.ops.neso.paged_attention(q, c, c, t, n, 0.1, 0.0, 0, None, weights)
            assert o.shape == q.shape and o.dtype == torch.float16
        kept, lens = torch.ops.neso.kv_evict(c, c.clone(), t, n, w, 24, 4, 2, None)
        assert kept.shape == (5, 2, 24) and kept.dtype == torch.int32 and lens.shape == (5,)
        x = e(5, 1000, dtype=torch.bfloat16)
        y = torch.ops.neso.process_logits(x, None, None, None, None, None, None, None, None, None)
        assert y.shape == x.shape and y.dtype == torch.bfloat16


def test_definition_of_attention():
    # two tokens, one page each, scores 0 and ln 3 at scale 1: weights 1/4 and 3/4
    k = torch.zeros(2, 1, 1, 64)
    v = torch.zeros(2, 1, 1, 64)
    k[0, 0, 0, 0], v[0, 0, 0, 0] = math.log(3.0), 4.0
    q = torch.zeros(1, 2, 64)
    q[0, :, 0] = 1.0
    table, n = torch.tensor([[1, 0]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    out, sums, _ = oracle.decode_attention(q, k, v, table, n, 1.0)
    assert out[0, 0, 0].item() == pytest.approx(3.0) and out[0, 0, 1].item() == 0.0
    assert sums[0, 0][0] == pytest.approx(0.5) and sums[0, 0][1] == pytest.approx(1.5)
    # the last token alone, capped, and a distance bias that evens the two out
    assert oracle.decode_attention(q, k, v, table, n, 1.0, window=1)[0][0, 0, 0].item() == pytest.approx(4.0)
    capped = oracle.decode_attention(q, k, v, table, n, 1.0, softcap=1.0)[0][0, 0, 0].item()
    s = math.tanh(math.log(3.0))
    assert capped == pytest.approx(4 * math.exp(s) / (1 + math.exp(s)))
    even = oracle.decode_attention(q, k, v, table, n, 1.0, slopes=torch.tensor([-math.log(3.0), 0.0], dtype=torch.float64))[0]
    assert even[0, 0, 0].item() == pytest.approx(2.0) and even[0, 1, 0].item() == pytest.approx(3.0)
    # a page outside the cache, and no token at all
    table[0, 1] = 2
    assert oracle.decode_attention(q, k, v, table, n, 1.0)[0][0, 0, 0].item() == 0.0
    assert bool((oracle.decode_attention(q, k, v, table, n * 0, 1.0)[0] == 0).all())


def test_definition_of_eviction_and_logits():
    w = torch.tensor([[[0.0, 5.0, 1.0, 1.0, math.nan, 0.0, 9.0]]])
    assert oracle.decode_evict(w, torch.tensor([7]), 4, 1, 1, 7) == [[[0, 1, 4, 6]]]
    assert oracle.decode_evict(w, torch.tensor([7]), 5, 1, 1, 7) == [[[0, 1, 2, 4, 6]]]  # a tie: the lower index
    assert oracle.decode_evict(w, torch.tensor([3]), 4, 1, 1, 7) == [[[0, 1, 2]]]
    x = torch.tensor([[2.0, -2.0, 1.0, 0.5]])
    y, _ = oracle.decode_logits(x, history=torch.tensor([[0, 1, 1, 9]]), history_lens=torch.tensor([4]),
                                prompt_lens=torch.tensor([1]), repetition=torch.tensor([2.0]), frequency=torch.tensor([0.25]),
                                presence=torch.tensor([0.5]), bias_ids=torch.tensor([[2, 2]]), bias=torch.tensor([[1.0, 2.0]]),
                                mask=torch.tensor([[7]]))
    assert y.tolist() == [[1.0, -5.0, 4.0, -math.inf]]
