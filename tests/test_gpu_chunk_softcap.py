"""Soft caps of attention of chunks: a capped score is as exact, relative to itself, as
32 bits hold it, however far below the cap it is.

Queries and keys have one element other than 0, so a score is one product.  A
capped score t = c tanh(s / c) then differs by
  2 u |t|  for the product and its scale,
  3 u |t|  for s / c (two roundings of the factor, one of the product; the
           relative change of tanh is at most that of its argument),
  8 u |t|  for the tanh (its exponential, sum and reciprocal off by 6 u in all where
           2 / (e^2x + 1) is at most 1.2 times the result, and that sum's rounding),
  2 u |t|  for c log2 e,
and its exponent, less the largest, by a rounding of the largest: 16 u of the largest |t|
together.  A probability by twice that and the exponential's own 4 u, the sums over n
keys by (n + 32) u."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle.serving import U
from serving import DTYPES, Cache, f64, i32, within
from test_gpu_chunk import SPLIT

pytestmark = pytest.mark.gpu


def check(dtype, D, news, had, cap, size, scale, seed, window=0):
    c = Cache([news + had], 1, D, 16, dtype, seed)
    n = news + had
    g = torch.Generator().manual_seed(seed)
    k = torch.zeros(c.k.shape)
    k[..., 0] = torch.randn(k.shape[:-1], generator=g)
    c.k = k.to(DTYPES[dtype]).cuda()
    q = torch.zeros(news, 2, D)
    q[..., 0] = size * torch.randn(news, 2, generator=g)
    q = q.to(DTYPES[dtype]).cuda()
    got = mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32([n]), i32([0, news]), softcap=cap, scale=scale, window=window)
    at = np.arange(n)
    kk, vv = (f64(p)[c.table[0, at // 16], 0, at % 16] for p in (c.k, c.v))
    want, slack = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(news):
        lo, hi = (max(0, had + t + 1 - window) if window else 0), had + t + 1
        for h in range(2):
            cap64 = np.float64(np.float32(cap))
            s = cap64 * np.tanh(f64(q)[t, h, 0] * kk[lo:hi, 0] * np.float64(np.float32(scale)) / cap64)
            p = np.exp(s - s.max())
            p /= p.sum()
            want[t, h] = p @ vv[lo:hi]
            slack[t, h] = p @ np.abs(vv[lo:hi]) * (2 * 16 * U * np.abs(s).max() + 4 * U + SPLIT[dtype] + (hi - lo + 32) * U)
    within(got, want, slack, (cap, size))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("cap", [1.0, 20.0, 30.0, 50.0, 1000.0, 1e5])
@pytest.mark.parametrize("size", [0.1, 1.0, 6.0])
def test_scores_far_below_the_cap(dtype, cap, size):
    announce("chunk soft cap", dtype, cap, size)
    check(dtype, 64, 40, 0, cap, size, 1.0, 7)


@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0])
@pytest.mark.parametrize("scale", [0.3, -0.3])
def test_scores_about_the_cap(cap, scale):
    """From a hundredth of the cap to many times it: where the forms of the tanh meet, and its ends."""
    announce("chunk soft cap all sizes", cap, scale)
    for ratio in (0.01, 0.3, 0.5, 0.6, 1.0, 4.0, 100.0):
        check("f32", 64, 33, 5, cap, ratio * cap / abs(scale), scale, 8)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D,news,had,window", [(64, 3, 3000, 0), (128, 140, 500, 0), (80, 200, 300, 0), (192, 70, 200, 0),
                                               (256, 70, 200, 0), (96, 150, 100, 60), (128, 1, 9000, 0)])
def test_long_caches(dtype, D, news, had, window):
    announce("chunk soft cap long", dtype, D, news, had, window)
    check(dtype, D, news, had, 50.0, 3.0, 1.0, 9, window)
