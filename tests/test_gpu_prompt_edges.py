"""The operators of prompts (rotation, rotated append, attention of chunks, logit
adjustments) at their edges: both ways into the library, capture after a reserve
alone, malformed starts, results joined from many workgroups, tables of edits
that are full, offsets past 32 bits.  Tolerances: those of their own tests."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
import test_gpu_adjust as adjust
import test_gpu_chunk as chunk
from helpers import announce
from serving import DTYPES, Cache, f64, i32

pytestmark = pytest.mark.gpu


def test_the_ctypes_path_gives_the_same(monkeypatch):
    from mlxcel_amd import ops

    announce("prompt operators ctypes")
    c = Cache([33, 5], 2, 64, 16, "f16", 81)
    starts, q = i32([0, 20, 23]), chunk.queries(23, 4, 64, "f16", 82)
    kv = chunk.queries(23, 2, 64, "f16", 83)
    table, lengths = i32(c.table), i32(c.lengths)
    positions, rows = i32([*range(13, 33), 2, 3, 40]), i32([0] * 20 + [1] * 3)
    inv, _ = mq.rotary_frequencies(64, scaling="bands", factor=8.0, original=8192)
    x = adjust.logits(3, 500, "f16", 84)
    a = adjust.on_gpu(adjust.case(3, 500, 40, 6, True, 85))

    def run():
        k, v = c.k.clone(), c.v.clone()
        return [mq.rotary(q, positions, inv, interleaved=True, factor=1.5),
                mq.rotary_append(q, kv, kv, k, v, table, positions, rows, inv, lengths=lengths, interleaved=True), k, v,
                mq.paged_attention_chunk(q, c.k, c.v, table, lengths, starts, window=9, softcap=20.0), mq.adjust_logits(x, **a)]

    want = run()
    monkeypatch.setattr(ops, "_native", ops._ctypes_only)
    for got, w in zip(run(), want):
        assert torch.equal(got.view(torch.int16), w.view(torch.int16))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_capture_after_a_reserve_alone(D):
    """131 MiB hold the partial results of every call."""
    announce("chunk reserve", D)
    news, had = [300, 1, 200], [2000, 9000, 0]
    c = Cache([a + b for a, b in zip(news, had)], 4, D, 16, "bf16", D)
    q, table, lengths, starts = chunk.queries(501, 32, D, "bf16", 5), i32(c.table), i32(c.lengths), i32(chunk.starts_of(news))
    want = mq.paged_attention_chunk(q, c.k, c.v, table, lengths, starts)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        mq.workspace_reserve(131 << 20)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = mq.paged_attention_chunk(q, c.k, c.v, table, lengths, starts)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        out.zero_()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_out_may_be_q(dtype):
    """Also where several workgroups read a tile's queries and one of them writes its results."""
    announce("chunk in place", dtype)
    news, had = [5, 40, 1], [6000, 0, 2000]
    c = Cache([a + b for a, b in zip(news, had)], 2, 128, 16, dtype, 6)
    q = chunk.queries(46, 8, 128, dtype, 7)
    args = i32(c.table), i32(c.lengths), i32(chunk.starts_of(news))
    want = mq.paged_attention_chunk(q, c.k, c.v, *args)
    for _ in range(3):
        mine = q.clone()
        assert mq.paged_attention_chunk(mine, c.k, c.v, *args, out=mine) is mine and torch.equal(mine, want)
    wide = torch.zeros(46, 8, 200, dtype=q.dtype, device="cuda")
    wide[..., 8:136] = q
    view = wide[..., 8:136]
    mq.paged_attention_chunk(view, c.k, c.v, *args, out=view)
    assert torch.equal(view, want) and not bool(wide[..., :8].any()) and not bool(wide[..., 136:].any())


def test_malformed_starts():
    """Starts out of range are cut to the tokens, descending ones leave a sequence nothing; the
    other sequences' rows are what they are with proper starts."""
    announce("chunk malformed starts")
    c = Cache([40, 7, 60], 2, 64, 16, "bf16", 3)
    q = chunk.queries(10, 4, 64, "bf16", 4)
    call = lambda starts: mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts))
    want = call([0, 3, 3, 10])
    assert torch.equal(call([-5, 3, 3, 100]), want)
    assert torch.equal(call([-2 ** 31, 3, 3, 2 ** 31 - 1]), want)
    both = call([0, 6, 4, 10])  # the second has none; rows 4 and 5 belong to two
    assert torch.equal(both[:4], call([0, 6, 6, 10])[:4]) and torch.equal(both[6:], call([0, 4, 4, 10])[6:])
    chunk.check(c, q, np.array([0, 3, 3, 10], np.int32), "bf16", got=want)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D,window", [(64, 0), (96, 0), (128, 0), (128, 5000), (192, 0), (256, 0)])
def test_results_joined_from_many_workgroups(dtype, D, window):
    """One head over 17000 keys: a hundred workgroups' results, in two steps of the join."""
    announce("chunk join", dtype, D, window)
    news, had = [2, 1], [17000, 300]
    c = Cache([a + b for a, b in zip(news, had)], 1, D, 16, dtype, D)
    q = chunk.queries(3, 3, D, dtype, 7)
    kw = dict(window=window) if window else {}
    first = chunk.check(c, q, chunk.starts_of(news), dtype, **kw)
    for _ in range(5):  # whoever is last
        assert torch.equal(mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(chunk.starts_of(news)), **kw),
                           first)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_every_token_in_the_history(dtype):
    """Whole stretches of a row edited: the lists are full; tokens twice, some with a bias, others with a bias alone."""
    announce("adjust full", dtype)
    V = 6200
    x = adjust.logits(2, V, dtype, 1)
    r = np.random.default_rng(2)
    h = np.stack([r.permutation(np.concatenate([np.arange(5000), np.arange(0, 5000, 3)])) for _ in range(2)]).astype(np.int32)
    ids = np.stack([r.permutation(np.concatenate([np.arange(4000, V), np.arange(4000, V)])) for _ in range(2)]).astype(np.int32)
    a = dict(history=h, prompts=np.int32([3000, 0]), repetition=np.float32([1.3, 0.9]), presence=np.float32([0.5, -0.5]),
             frequency=np.float32([0.25, 1.5]), bias_ids=ids, bias=(r.random(ids.shape) * 8 - 4).astype(np.float32))
    first = mq.adjust_logits(x, **adjust.on_gpu(a))
    adjust.check(x, a, first)
    for _ in range(3):
        assert torch.equal(mq.adjust_logits(x, **adjust.on_gpu(a)), first)
    y = x.clone()  # in place
    assert mq.adjust_logits(y, out=y, **adjust.on_gpu(a)) is y and torch.equal(y, first)


def test_edits_that_give_zero_and_nan():
    """New logits whose bits are 0, or a NaN of any bits, are no untouched ones."""
    announce("adjust zero")
    for dtype in DTYPES:
        x = adjust.logits(1, 40, dtype, 3)
        bias = np.float32([0, 0, np.nan, 0])
        bias[0], bias[1] = -float(x[0, 5]), np.inf
        bias[3:].view(np.uint32)[0] = 0xFFFFFFFF  # the NaN whose bits are all ones
        got = mq.adjust_logits(x, bias_ids=i32([[5, 6, 7, 8]]), bias=torch.from_numpy(bias[None].copy()).cuda())
        assert float(got[0, 5]) == 0 and float(got[0, 6]) == float("inf") and bool(got[0, 7:9].isnan().all())
        assert torch.equal(got[0, 9:], x[0, 9:])


def test_rows_past_32_bits():
    """14300 rows of 151936: 2.2e9 logits, in place."""
    announce("adjust far rows")
    T, V = 14300, 151936
    x = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    few = [0, 7000, 14134, 14135, T - 1]
    rows = adjust.logits(len(few), V, "bf16", 4)
    x[few] = rows
    a = adjust.case(T, V, 6, 2, False, 5)
    assert mq.adjust_logits(x, out=x, **adjust.on_gpu(a)) is x
    adjust.check(rows, {k: v[few] for k, v in a.items()}, x[few])
