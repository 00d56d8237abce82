"""Attention of chunks where scores are so large that 32 bits hold them in steps
of 1 and more: what is finite stays finite.

Queries and keys have one element other than 0, whole numbers of at most 10 bits
times a power of two, so a score is exact; keys come in two values of opposite
sign.  All keys but those of the largest score then have probability 0, and those have
equal ones: the result is the mean of their values.

Tolerance: the sums over n keys, (n + 32) u of the mean of |v|, and SPLIT's loss
of a probability; where a tile's keys may be cut over workgroups, equal scores of two
parts may be weighed differently by a rounding of the score (here 1 or more in the
exponent), and the result only has to lie between the values that it is made of."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle.serving import U
from serving import DTYPES, Cache, f64, i32, within
from test_gpu_chunk import SPLIT

pytestmark = pytest.mark.gpu

# powers of two of a query's and a key's element, each times 512 .. 1023
POWERS = {"f16": [(3, 3), (4, 5), (6, 6)], "bf16": [(0, 1), (2, 3), (6, 6), (20, 30), (40, 40)],
          "f32": [(0, 1), (2, 3), (6, 6), (20, 30), (40, 40)]}


def large(news, had, Hq, Hkv, D, dtype, powers, seed):
    """(cache, queries): whole numbers of 512 .. 1020 in steps of 4 (bfloat16: 8 bits) times powers of two."""
    c = Cache([a + b for a, b in zip(news, had)], Hkv, D, 16, dtype, seed)
    r = np.random.default_rng(seed)
    x = 4.0 * r.integers(128, 256, c.pages) * 2.0 ** powers[1]
    k = torch.zeros(c.k.shape, dtype=torch.float64)
    for b, row in enumerate(c.table):
        for j, p in enumerate(row):  # one size a sequence, its sign positive at every seventh place
            sign = np.where((16 * j + np.arange(16)) % 7 == 0, 1.0, -1.0)
            k[p, :, :, 0] = torch.from_numpy(x[b] * sign)
    c.k = k.to(DTYPES[dtype]).cuda()
    q = torch.zeros(sum(news), Hq, D, dtype=torch.float64)
    q[..., 0] = torch.from_numpy(4.0 * r.integers(128, 256, (sum(news), Hq)) * 2.0 ** powers[0] * r.choice([-1, 1], (sum(news), Hq)))
    return c, q.to(DTYPES[dtype]).cuda()


def means(c, q, starts):
    """For each row: the mean of the values of the largest score, of their sizes, the least, the largest, the keys
    seen, whether that score is positive."""
    T, Hq, D = q.shape
    q, v, k = f64(q), f64(c.v), f64(c.k)
    mean, size, lo, hi = (np.zeros((T, Hq, D)) for _ in range(4))
    seen, positive = np.zeros((T, 1, 1)), np.zeros((T, Hq, 1), bool)
    for b, length in enumerate(c.lengths):
        at = np.arange(length)
        for h in range(Hq):
            kk, vv = (p[c.table[b, at // 16], h // (Hq // c.Hkv), at % 16] for p in (k, v))
            for t in range(starts[b], starts[b + 1]):
                n = length - (starts[b + 1] - t) + 1
                s = q[t, h, 0] * kk[:n, 0]
                best = vv[:n][s == s.max()]
                mean[t, h], size[t, h], lo[t, h], hi[t, h] = best.mean(0), np.abs(best).mean(0), best.min(0), best.max(0)
                seen[t], positive[t, h] = n, s.max() > 0
    return mean, size, lo, hi, seen, positive


def call(c, q, starts, **kw):
    return mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts), **{"scale": 1.0, **kw})


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 80, 128, 192, 256])
def test_short_sequences(dtype, D):
    """Tiles that no workgroups share."""
    news, had = [60, 1, 33, 5], [0, 200, 90, 250]
    starts = np.concatenate([[0], np.cumsum(news)])
    for n, powers in enumerate(POWERS[dtype]):
        announce("chunk large scores", dtype, D, powers)
        c, q = large(news, had, 4, 2, D, dtype, powers, D + n)
        got = call(c, q, starts)
        mean, size, _, _, seen, positive = means(c, q, starts)
        within(got, mean, size * ((seen + 32) * U + SPLIT[dtype]), powers)
        # sinks that are nothing beside such scores, and all there is beside negative ones
        got = call(c, q, starts, sinks=torch.tensor([3.0, -3.0, 0.0, 8.0], device="cuda"))
        m, s = np.where(positive, mean, 0), np.where(positive, size, 0)
        within(got, m, s * ((seen + 32) * U + SPLIT[dtype]), powers)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 128, 256])
def test_long_sequences(dtype, D):
    """Steps without masks and tiles that workgroups share."""
    news, had = [150, 3], [900, 3000]
    starts = np.concatenate([[0], np.cumsum(news)])
    for n, powers in enumerate(POWERS[dtype]):
        announce("chunk large scores long", dtype, D, powers)
        c, q = large(news, had, 2, 1, D, dtype, powers, D + n)
        got = f64(call(c, q, starts))
        mean, size, lo, hi, seen, _ = means(c, q, starts)
        info = torch.finfo(DTYPES[dtype])
        slack = size * ((seen + 32) * U + SPLIT[dtype]) + info.eps / 2 * np.maximum(np.abs(lo), np.abs(hi)) + info.tiny
        assert ((got >= lo - slack) & (got <= hi + slack)).all(), powers


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_large_cap(dtype):
    """Scores of either end of a soft cap of 2^40: ties, whose probabilities are equal."""
    announce("chunk large cap", dtype)
    news, had = [40, 9], [10, 130]
    starts = np.concatenate([[0], np.cumsum(news)])
    c, q = large(news, had, 4, 2, 64, dtype, (6, 6), 5)
    got = call(c, q, starts, softcap=2.0 ** 40, scale=2.0 ** 30)
    mean, size, _, _, seen, _ = means(c, q, starts)
    within(got, mean, size * ((seen + 32) * U + SPLIT[dtype]))
