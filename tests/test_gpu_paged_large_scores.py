"""Attention of single tokens where scores are so large that 32 bits hold them in
steps of 1 and more: what is finite stays finite.  The caches, queries and tolerances are
those of the chunks' test."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle.serving import U
from serving import DTYPES, f64, i32, within
from test_gpu_chunk_large_scores import POWERS, large, means

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("Hq,D", [(4, 64), (2, 128), (4, 80), (4, 256)])
def test_large_scores(dtype, Hq, D):
    had = list(range(1, 70, 3)) + [250]
    B = len(had)
    for n, powers in enumerate(POWERS[dtype]):
        announce("paged large scores", dtype, Hq, D, powers)
        c, q = large([1] * B, had, Hq, 2, D, dtype, powers, D + n)
        got = mq.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lengths), scale=1.0)
        mean, size, _, _, seen, _ = means(c, q, np.arange(B + 1))
        # of a probability at most 2^-24 of itself is left out, or 2^-39 of the largest
        within(got, mean, size * ((seen + 32) * U + 2.0 ** -24), powers)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_long_caches(dtype):
    """Caches that workgroups share: between the values of the largest score."""
    had = [3000, 9000, 700]
    for n, powers in enumerate(POWERS[dtype]):
        announce("paged large scores long", dtype, powers)
        c, q = large([1] * 3, had, 4, 1, 64, dtype, powers, n)
        got = f64(mq.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lengths), scale=1.0))
        _, size, lo, hi, seen, _ = means(c, q, np.arange(4))
        info = torch.finfo(DTYPES[dtype])
        slack = size * ((seen + 32) * U + 2.0 ** -24) + info.eps / 2 * np.maximum(np.abs(lo), np.abs(hi)) + info.tiny
        assert ((got >= lo - slack) & (got <= hi + slack)).all(), powers
