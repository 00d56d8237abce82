"""Attention of chunks over caches that take the kernel's other ways in: heads
narrower than the kernel over steps without masks and tiles that workgroups share, pools whose
rows are not aligned to 16 bytes, keys and values of different strides.

Tolerance: as in the chunks' own tests."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from serving import DTYPES, Cache, i32
from test_gpu_chunk import check, queries, starts_of
from test_gpu_chunk_values import check_but

pytestmark = pytest.mark.gpu


def split_strides(c, which):
    """The same pools, keys or values with tokens before heads in memory."""
    turned = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    if which == "keys":
        c.k = turned(c.k)
    else:
        c.v = turned(c.v)
    assert c.k.stride() != c.v.stride()
    return c


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [8, 40, 56, 72, 80, 88, 104, 136, 160, 200, 232])
@pytest.mark.parametrize("window", [0, 500])
def test_narrow_heads(dtype, D, window):
    """160 new tokens of 1200: steps without masks; 3 of 2500 on one head of keys: many workgroups a tile."""
    announce("chunk narrow heads", dtype, D, window)
    news, had = [160, 3], [1040, 2497]
    c = Cache([a + b for a, b in zip(news, had)], 1, D, 16, dtype, D)
    check(c, queries(sum(news), 2, D, dtype, 1), starts_of(news), dtype, window=window)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 80, 128, 136, 256])
@pytest.mark.parametrize("window", [0, 100])
def test_rows_that_are_not_aligned(dtype, D, window):
    """Keys and values in one allocation, rows two elements apart."""
    announce("chunk unaligned", dtype, D, window)
    news, had = [150, 2, 33], [600, 1500, 0]
    c = Cache([a + b for a, b in zip(news, had)], 2, D, 16, dtype, D, layout="both")
    check(c, queries(sum(news), 4, D, dtype, 2), starts_of(news), dtype, window=window)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_keys_and_values_of_different_strides(dtype, D, which):
    announce("chunk strides of its own", dtype, D, which)
    news, had = [150, 2, 33], [600, 1500, 0]
    c = split_strides(Cache([a + b for a, b in zip(news, had)], 2, D, 16, dtype, D), which)
    check(c, queries(sum(news), 4, D, dtype, 3), starts_of(news), dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("layout", ["both", "keys", "values"])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_values_that_are_not_finite(dtype, layout, D):
    """The slow way over the same pools: a value at a key that part of the new tokens see."""
    announce("chunk layouts values", dtype, layout, D)
    news, had, at = [60, 5], [300, 700], 330
    c = Cache([a + b for a, b in zip(news, had)], 2, D, 16, dtype, D, layout="both" if layout == "both" else "pages")
    if layout != "both":
        c = split_strides(c, layout)
    q, starts = queries(65, 4, D, dtype, 4), starts_of(news)
    v = c.v[int(c.table[0, at // 16]), :, at % 16, 3]
    clean, was = c.v.clone(), v.clone()
    v[:] = float("inf")
    got = mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts))
    hit = np.arange(65) >= at - 300
    check_but(c, clean, q, starts, dtype, got, hit & (np.arange(65) < 60), [3])
    v[:] = was
