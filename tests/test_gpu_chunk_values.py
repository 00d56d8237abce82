"""Values that are not finite in attention of chunks: they reach the tokens that
see their key, wherever it lies, and no other token, sequence or column."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, Cache, f64, i32, within
from test_gpu_chunk import SPLIT, queries, starts_of

pytestmark = pytest.mark.gpu

INF = float("inf")


def call(c, q, starts, **kw):
    return mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts), **kw)


def place(c, b, at):
    return int(c.table[b, at // c.page]), slice(None), at % c.page


def check_but(c, clean_v, q, starts, dtype, got, hit, columns, window=0, peaked=0):
    """Rows in `hit` are not finite in `columns`; all else is what finite values there give."""
    want, slack, live = ref.chunk_attention(f64(q), f64(c.k), f64(clean_v), c.table, c.lengths, starts,
                                            np.float64(np.float32(q.shape[-1] ** -0.5)), window=window, split=SPLIT[dtype])
    g = got.clone()
    bad = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    for col in columns:
        bad[torch.from_numpy(hit).cuda(), :, col] = True
    assert not bool(torch.isfinite(g[bad]).any())
    g[bad] = torch.from_numpy(want).cuda()[bad].to(g.dtype)
    within(g[torch.from_numpy(live).cuda()], want[live], slack[live])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [float("nan"), INF, -INF])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 1), (80, 4, 2), (96, 2, 2), (128, 4, 2), (192, 2, 1), (256, 4, 2), (200, 3, 1)])
def test_one_value(dtype, bad, D, Hq, Hkv):
    """At keys before the new tokens, among them, in masked blocks and in others, over steps without masks
    and joined tiles: one column, all heads."""
    news, had = [140, 2, 60], [500, 700, 0]
    starts = starts_of(news)
    c = Cache([a + b for a, b in zip(news, had)], Hkv, D, 16, dtype, D)
    q = queries(sum(news), Hq, D, dtype, 3)
    clean = c.v.clone()
    for b, at, col in ((0, 0, 0), (0, 333, D - 1), (0, 520, D // 2), (0, 639, 7), (1, 5, 3), (1, 700, 33), (2, 31, D - 8), (2, 59, 1)):
        announce("chunk values", dtype, bad, D, b, at)
        c.v = clean.clone()
        c.v[place(c, b, at) + (col,)] = bad
        hit = np.zeros(len(q), bool)
        hit[starts[b] + max(0, at - had[b]):starts[b + 1]] = True
        check_but(c, clean, q, starts, dtype, call(c, q, starts), hit, [col])
        if b == 0:  # and a window that leaves the key behind
            hit = np.zeros(len(q), bool)
            hit[max(0, at - had[b]):max(0, min(news[0], at - had[0] + 50))] = True
            check_but(c, clean, q, starts, dtype, call(c, q, starts, window=50), hit, [col], window=50)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_underflowed_probabilities(dtype, D):
    """A key that a token sees with a probability of 0 in 32 bits: an infinite value makes its column infinite or NaN,
    in the token's own block and in one before it, and however a prompt is cut."""
    news, had = 70, 100
    c = Cache([news + had], 1, D, 16, dtype, D)
    q = queries(news, 2, D, dtype, 4)
    q[..., 0] = 8.0
    for at, col in ((20, 5), (101, 9), (130, 0), (165, D - 1)):
        clean_k, clean_v = c.k, c.v
        c.k, c.v = c.k.clone(), c.v.clone()
        c.k[place(c, 0, at) + (0,)] = -8000.0  # scores some 64000 / sqrt(D) below the others
        finite = c.v.clone()
        c.v[place(c, 0, at) + (col,)] = INF
        hit = np.arange(news) + had >= at
        for cut in ((0, news), (0, 1, 31, news), (0, 30, 62, news), (0, 65, news)):
            announce("chunk underflow", dtype, D, at, cut)
            for a, b in zip(cut[:-1], cut[1:]):
                lengths = c.lengths
                c.lengths = np.int32([had + b])
                check_but(c, finite, q[a:b], np.int32([0, b - a]), dtype, call(c, q[a:b], [0, b - a]), hit[a:b], [col])
                c.lengths = lengths
        c.k, c.v = clean_k, clean_v


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [float("nan"), INF])
@pytest.mark.parametrize("D", [64, 128, 192])
def test_keys_of_minus_infinity(dtype, bad, D):
    """Keys whose score is -inf have no part in the result, whatever their values are."""
    news, had = 70, 300
    c = Cache([news + had], 1, D, 16, dtype, D)
    q = queries(news, 2, D, dtype, 4)
    q[..., 0] = 1.0
    for at in (20, 200, 301, 350):
        c.k[place(c, 0, at) + (0,)] = -INF
    finite = c.v.clone()
    for at in (20, 200, 301, 350):
        announce("chunk -inf keys", dtype, bad, D, at)
        c.v = finite.clone()
        c.v[place(c, 0, at)] = bad
        check_but(c, finite, q, np.int32([0, news]), dtype, call(c, q, [0, news]), np.zeros(news, bool), [])
