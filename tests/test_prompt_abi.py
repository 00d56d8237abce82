"""CPU checks of rotary positions, rotated appends, attention of chunks and
logit adjustments: refused arguments (only calls that fail before any device
work), the frequencies, the wrappers' refusals, the 64-bit forms."""
import ctypes
import math

import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from mlxcel_amd import _lib
from oracle import serving as ref
from test_serving_abi import BF, EINVAL, EUNSUPPORTED, F16, F32, F64, I32, I64, arr, have, refused

UINT32 = _lib.UINT32


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def args_of(base, change):
    return [have(*v) if isinstance(v, tuple) else v for v in {**base, **change}.values()]


ATTN = dict(q=((12, 8, 64), BF), k=((9, 2, 16, 64), BF), v=((9, 2, 16, 64), BF), table=((2, 5), I32), lengths=((2,), I32),
            starts=((3,), I32), sinks=None, scale=0.125, softcap=0.0, window=0, out=((12, 8, 64), BF))


@pytest.mark.parametrize("change,code,text", [
    (dict(q=((12, 8), BF)), EINVAL, "q must have 3 dimensions"),
    (dict(q=((12, 8, 64), F64)), EINVAL, "bfloat16, float16 or float32 but is float64"),
    (dict(k=((9, 2, 16, 64), F16)), EINVAL, "k_pool must be bfloat16"),
    (dict(v=((9, 2, 8, 64), BF)), EINVAL, "v_pool must have shape"),
    (dict(q=((12, 7, 64), BF)), EINVAL, "query heads (7)"),
    (dict(q=((12, 8, 72), BF)), EINVAL, "one head width"),
    (dict(table=((3, 5), I32)), EINVAL, "as many rows"),
    (dict(table=((2, 5), I64)), EINVAL, "table must be int32"),
    (dict(table=((2, 1 << 27), I32)), EUNSUPPORTED, "too wide"),
    (dict(starts=((2,), I32)), EINVAL, "one entry more"),
    (dict(starts=((3,), I64)), EINVAL, "starts must be int32"),
    (dict(starts=((3,), I32, (2,))), EUNSUPPORTED, "starts must be contiguous"),
    (dict(sinks=((7,), F32)), EINVAL, "sinks must have shape"),
    (dict(scale=float("inf")), EINVAL, "scale"),
    (dict(softcap=-1.0), EINVAL, "softcap"),
    (dict(window=-1), EINVAL, "window"),
    (dict(out=((12, 8, 64), F32)), EINVAL, "out must have shape"),
    (dict(k=((9, 2, 16, 64), BF, (2048, 1024, 1, 16))), EUNSUPPORTED, "last axis must be contiguous"),
    (dict(k=((9, 2, 0, 64), BF), v=((9, 2, 0, 64), BF)), EINVAL, "no pages"),
    (dict(q=((12, 8, 60), BF), k=((9, 2, 16, 60), BF), v=((9, 2, 16, 60), BF), out=((12, 8, 60), BF)), EUNSUPPORTED,
     "multiple of 8"),
    (dict(q=((12, 8, 264), BF), k=((9, 2, 16, 264), BF), v=((9, 2, 16, 264), BF), out=((12, 8, 264), BF)), EUNSUPPORTED,
     "up to 256"),
])
def test_paged_attention_chunk(lib, change, code, text):
    refused(lib, "mlxq_paged_attention_chunk", code, text, *args_of(ATTN, change))


ROTARY = dict(x=((5, 3, 16), BF), positions=((5,), I32), inv_freq=((8,), F32), interleaved=False, factor=1.0,
              out=((5, 3, 16), BF))


@pytest.mark.parametrize("change,code,text", [
    (dict(x=((5, 16), BF)), EINVAL, "3 dimensions"),
    (dict(x=((5, 3, 16), I32)), EINVAL, "bfloat16, float16 or float32"),
    (dict(positions=((4,), I32)), EINVAL, "positions must have shape"),
    (dict(positions=((5,), I64)), EINVAL, "positions must be int32"),
    (dict(inv_freq=((9,), F32)), EINVAL, "9 pairs but a head has 16"),
    (dict(inv_freq=((8,), BF)), EINVAL, "inv_freq must be float32"),
    (dict(inv_freq=((8,), F32, (2,))), EUNSUPPORTED, "inv_freq must be contiguous"),
    (dict(factor=float("nan")), EINVAL, "factor"),
    (dict(out=((5, 3, 16), F16)), EINVAL, "out must have shape"),
    (dict(x=((5, 3, 4104), BF), out=((5, 3, 4104), BF)), EUNSUPPORTED, "at most 4096"),
    (dict(x=((5, 40000, 16), BF), out=((5, 40000, 16), BF)), EUNSUPPORTED, "at most 32768 heads"),
    (dict(x=((1 << 31, 1, 16), BF, (0, 16, 1)), positions=((1 << 31,), I32), out=((1 << 31, 1, 16), BF)), EUNSUPPORTED,
     "too large"),
])
def test_rotary(lib, change, code, text):
    refused(lib, "mlxq_rotary", code, text, *args_of(ROTARY, change))


APPEND = dict(q=((3, 4, 8), BF), k=((3, 2, 8), BF), v=((3, 2, 8), BF), kp=((20, 2, 16, 8), BF), vp=((20, 2, 16, 8), BF),
              table=((4, 6), I32), positions=((3,), I32), rows=((3,), I32), lengths=None, inv_freq=((4,), F32),
              interleaved=True, factor=1.0, out=((3, 4, 8), BF))


@pytest.mark.parametrize("change,code,text", [
    (dict(q=((2, 4, 8), BF)), EINVAL, "same tokens and width"),
    (dict(k=((3, 2, 8), F16)), EINVAL, "k must be bfloat16"),
    (dict(v=((3, 1, 8), BF)), EINVAL, "v must have shape"),
    (dict(kp=((20, 3, 16, 8), BF), vp=((20, 3, 16, 8), BF)), EINVAL, "same heads and width"),
    (dict(vp=((20, 2, 8, 8), BF)), EINVAL, "v_pool must have shape"),
    (dict(kp=((20, 2, 16, 8), F32)), EINVAL, "k_pool must be bfloat16"),
    (dict(positions=((4,), I32)), EINVAL, "positions must have shape"),
    (dict(rows=((3,), I64)), EINVAL, "rows must be int32"),
    (dict(lengths=((3,), I32)), EINVAL, "lengths must have shape"),
    (dict(inv_freq=((5,), F32)), EINVAL, "5 pairs"),
    (dict(factor=float("inf")), EINVAL, "factor"),
    (dict(out=((3, 2, 8), BF)), EINVAL, "out must have shape"),
    (dict(kp=((20, 2, 16, 8), BF, (256, 128, 1, 16))), EUNSUPPORTED, "last axis must be contiguous"),
    (dict(kp=((0, 2, 16, 8), BF), vp=((0, 2, 16, 8), BF)), EINVAL, "no pages"),
    (dict(table=((4, 1 << 27), I32)), EUNSUPPORTED, "too wide"),
])
def test_rotary_append(lib, change, code, text):
    refused(lib, "mlxq_rotary_append", code, text, *args_of(APPEND, change))


ADJUST = dict(x=((3, 100), BF), history=((3, 7), I32), lengths=None, prompts=None, rep=None, pres=None, freq=None, ids=None,
              bias=None, mask=None, out=((3, 100), BF))


@pytest.mark.parametrize("change,code,text", [
    (dict(x=((100,), BF)), EINVAL, "2 dimensions"),
    (dict(x=((3, 100), I32)), EINVAL, "bfloat16, float16 or float32"),
    (dict(history=((2, 7), I32)), EINVAL, "one row"),
    (dict(history=((3, 7), I64)), EINVAL, "history must be int32"),
    (dict(history=((3, 7), I32, (7, 2))), EUNSUPPORTED, "rows must be contiguous"),
    (dict(lengths=((2,), I32)), EINVAL, "history_lengths must have shape"),
    (dict(rep=((3,), BF)), EINVAL, "repetition must be float32"),
    (dict(pres=((3, 1), F32)), EINVAL, "1 dimensions"),
    (dict(freq=((4,), F32)), EINVAL, "frequency must have shape"),
    (dict(history=None, prompts=((3,), I32)), EINVAL, "prompts needs a history"),
    (dict(history=None, freq=((3,), F32)), EINVAL, "frequency needs a history"),
    (dict(ids=((3, 2), I32)), EINVAL, "go together"),
    (dict(bias=((3, 2), F32)), EINVAL, "go together"),
    (dict(ids=((3, 2), I32), bias=((3, 3), F32)), EINVAL, "bias must have shape"),
    (dict(mask=((3, 3), I32)), EINVAL, "mask must have shape"),
    (dict(mask=((3, 4), UINT32)), EINVAL, "mask must be int32"),
    (dict(out=((3, 100), F32)), EINVAL, "out must have shape"),
    (dict(x=((1, (1 << 30) + 8), BF), history=None, out=((1, (1 << 30) + 8), BF)), EUNSUPPORTED, "too long"),
    (dict(x=((1 << 30, 100), BF), history=None, out=((1 << 30, 100), BF)), EUNSUPPORTED, "too many logits"),
    (dict(history=((3, (1 << 30) + 1), I32)), EUNSUPPORTED, "too long"),
    (dict(ids=((3, 1 << 31), I32), bias=((3, 1 << 31), F32)), EUNSUPPORTED, "too long"),
])
def test_adjust_logits(lib, change, code, text):
    refused(lib, "mlxq_adjust_logits", code, text, *args_of(ADJUST, change))


def test_data_pointers(lib):
    a = {k: have(*v) if isinstance(v, tuple) else v for k, v in ATTN.items()}
    refused(lib, "mlxq_paged_attention_chunk", EINVAL, "starts has no data", *{**a, "starts": arr((3,), I32)}.values())
    refused(lib, "mlxq_paged_attention_chunk", EINVAL, "not aligned",
            *{**a, "q": have((12, 8, 64), BF, None, 4097)}.values())
    refused(lib, "mlxq_rotary", EINVAL, "must not be NULL",
            *{k: None if k == "inv_freq" else have(*v) if isinstance(v, tuple) else v for k, v in ROTARY.items()}.values())


# ---- frequencies --------------------------------------------------------------------


def close(got, want):
    """A 32-bit rounding, and 64-bit noise next to a border between two values."""
    np.testing.assert_allclose(got.numpy().astype(np.float64), want, rtol=2.0 ** -24 * (1 + 1e-6))


@pytest.mark.parametrize("dims,base", [(2, 10000.0), (64, 10000.0), (80, 500000.0), (128, 1e6)])
def test_frequencies(dims, base):
    plain = base ** (-np.arange(0, dims, 2) / dims)
    got, by = mq.rotary_frequencies(dims, base, device="cpu")
    assert got.dtype == torch.float32 and got.shape == (dims // 2,) and by == 1
    close(got, plain)
    close(mq.rotary_frequencies(dims, base, scaling="linear", factor=4.0, device="cpu")[0], plain / 4)
    if dims > 2:
        close(mq.rotary_frequencies(dims, base, scaling="base", factor=8.0, device="cpu")[0],
              (base * 8.0 ** (dims / (dims - 2))) ** (-np.arange(0, dims, 2) / dims))
    # bands, by wavelengths
    wave = 2 * math.pi / plain
    want = np.where(wave > 8192 / 1.0, plain / 8, plain)
    mid = (wave <= 8192 / 1.0) & (wave >= 8192 / 4.0)
    part = (8192 / wave - 1.0) / (4.0 - 1.0)
    want = np.where(mid, (1 - part) * plain / 8 + part * plain, want)
    close(mq.rotary_frequencies(dims, base, scaling="bands", factor=8.0, original=8192, device="cpu")[0], want)
    # ramp, by the pairs' numbers
    at = lambda turns: dims * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base))
    first, last = max(math.floor(at(32)), 0), min(math.ceil(at(1)), dims - 1)
    ramp = np.clip((np.arange(dims // 2) - first) / max(last - first, 0.001), 0, 1)
    got, by = mq.rotary_frequencies(dims, base, scaling="ramp", factor=16.0, original=4096, device="cpu")
    close(got, plain / 16 * ramp + plain * (1 - ramp))
    assert by == np.float32(0.1 * math.log(16.0) + 1)


@pytest.mark.parametrize("change,text", [
    (dict(dims=0), "dims"), (dict(dims=7), "dims"), (dict(base=1.0), "base"), (dict(base=float("inf")), "base"),
    (dict(scaling="none"), "scaling"), (dict(scaling="linear", factor=0.5), "factor"),
    (dict(scaling="base", dims=2, factor=2.0), "4 dims"), (dict(scaling="bands", factor=2.0), "original"),
    (dict(scaling="bands", factor=2.0, original=100.0, low=4.0), "low"),
    (dict(scaling="ramp", factor=2.0, original=float("nan")), "original"),
])
def test_frequencies_refused(change, text):
    kw = {"dims": 8, "device": "cpu", **change}
    with pytest.raises(ValueError, match=text):
        mq.rotary_frequencies(kw.pop("dims"), **kw)


def test_frequencies_of_unknown_scalings_and_null(lib):
    out, by = (ctypes.c_float * 4)(), ctypes.c_float()
    assert lib.mlxq_rotary_frequencies(8, 1e4, 5, 2.0, 100.0, 1.0, 4.0, out, ctypes.byref(by)) == EINVAL
    assert lib.mlxq_rotary_frequencies(8, 1e4, 0, 2.0, 100.0, 1.0, 4.0, None, ctypes.byref(by)) == EINVAL


# ---- wrappers and 64-bit forms ------------------------------------------------------


def test_wrappers_refuse_tensors_off_the_device():
    x, i = torch.zeros(2, 2, 8), torch.zeros(2, dtype=torch.int32)
    pool, inv = torch.zeros(1, 2, 4, 8), torch.zeros(4)
    for f in (lambda: mq.paged_attention_chunk(x, pool, pool, i[:, None], i, i), lambda: mq.rotary(x, i, inv),
              lambda: mq.rotary_append(x, x, x, pool, pool, i[:, None], i, i, inv), lambda: mq.adjust_logits(x[0])):
        with pytest.raises(ValueError, match="HIP device"):
            f()


def test_chunk_form():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((6, 4, 8), (5, 2, 4, 8), (5, 2, 4, 8)))
    table = np.array([[3, 0, 4], [1, 2, 0]])
    got, slack, live = ref.chunk_attention(q.numpy(), k.numpy(), v.numpy(), table, [10, 2], np.array([1, 5, 6]), 0.5)
    assert live.tolist() == [False] + [True] * 5
    flat = lambda t: t[table[0]].transpose(0, 1).reshape(2, 12, 8)[:, :10].repeat_interleave(2, 0)
    mask = torch.ones(10, 10, dtype=torch.bool).tril()[6:]
    want = torch.nn.functional.scaled_dot_product_attention(q[1:5].transpose(0, 1), flat(k), flat(v), attn_mask=mask,
                                                            scale=0.5).transpose(0, 1)
    np.testing.assert_allclose(got[1:5], want.numpy(), rtol=1e-12)
    assert 0 < slack[1:].max() < 1e-4 and not slack[0].any()
    got, _, _ = ref.chunk_attention(q.numpy(), k.numpy(), v.numpy(), table, [2, 9], np.array([0, 4, 6]), 0.5, window=1)
    assert not got[:2].any()
    np.testing.assert_allclose(got[2], v[3, :, 0].repeat_interleave(2, 0).numpy(), rtol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_form(interleaved):
    g = np.random.default_rng(1)
    x, pos, f = g.normal(size=(3, 2, 10)), np.array([0, 5, -70]), np.float32([1, 0.3, 0.01])
    y, slack = ref.rotary(x, pos, f, interleaved, 2.0)
    for t in range(3):
        for i in range(3):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, 3 + i)
            z = (x[t, :, a] + 1j * x[t, :, b]) * 2 * np.exp(1j * pos[t] * np.float64(f[i]))
            np.testing.assert_allclose(y[t, :, a] + 1j * y[t, :, b], z, rtol=1e-11)
    assert np.array_equal(y[..., 6:], x[..., 6:]) and not slack[..., 6:].any() and (slack[..., :6] > 0).all()
    back, _ = ref.rotary(y, -pos, f, interleaved, 0.5)
    np.testing.assert_allclose(back, x, rtol=1e-11)


def test_adjust_form():
    x = np.array([[2.0, -2.0, 1.0, 0.5, 3.0]])
    y, slack, changed = ref.adjust_logits(x, np.array([[1, 0, 4, 4, 9, 2]]), np.array([5]), np.array([2]), np.array([2.0]),
                                          np.array([0.5]), np.array([0.25]), np.array([[3, 0, 3]]),
                                          np.array([[1.0, 10.0, 2.0]]), np.array([[0b10111 | 1 << 31]], np.int64).astype(np.int32))
    np.testing.assert_allclose(y, [[11.0, -4.0, 1.0, -np.inf, 1.5 - 1.0]])
    assert changed.tolist() == [[True, True, False, True, True]] and slack[0, 2] == 0
