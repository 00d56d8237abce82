"""Tiles that one workgroup works out one after the other: what is not finite in one
changes nothing in the next, also where the head is narrower than the kernel."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from serving import DTYPES, Cache, i32
from test_gpu_chunk import queries, starts_of

pytestmark = pytest.mark.gpu


def call(c, q, starts, **kw):
    return mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts), **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [72, 80, 88, 40, 104, 64])
def test_another_sequences_values_change_no_bit(dtype, D):
    """Workgroups take tiles of several sequences one after the other; some of these have infinite values."""
    announce("chunk neighbours", dtype, D)
    B, Hkv = 1200, 2
    r = np.random.default_rng(D)
    news, had = r.integers(9, 24, B), r.integers(0, 60, B)
    c = Cache((news + had).tolist(), Hkv, D, 16, dtype, D)
    starts = starts_of(news)
    q = queries(int(news.sum()), 4 * Hkv, D, dtype, 5)
    want = call(c, q, starts)
    clean = c.v.clone()
    good = torch.ones(len(q), dtype=torch.bool, device="cuda")
    for b in range(0, B, 10):
        for p in c.table[b, :-(-int(news[b] + had[b]) // 16)]:
            c.v[int(p)] = float("inf")
        good[starts[b]:starts[b + 1]] = False
    got = call(c, q, starts)
    assert not bool(torch.isfinite(got[~good]).any())
    assert torch.equal(got[good], want[good])
    c.v = clean
