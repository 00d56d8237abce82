"""Keys that are not finite in attention of chunks: what the tokens that see them get.

A NaN, or an infinite element that makes a score of +inf, gives a row of NaN (inf - inf); one that
makes a score of -inf leaves the key out."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, Cache, f64, i32, within
from test_gpu_chunk import SPLIT, queries, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D,window", [(64, 0), (64, 40), (80, 0), (128, 0), (256, 0), (192, 40)])
def test_keys_that_are_not_finite(dtype, bad, D, window):
    news, had = [140, 3], [400, 900]
    starts = starts_of(news)
    q = queries(143, 4, D, dtype, 3)
    for b, at in ((0, 10), (0, 390), (0, 401), (0, 470), (1, 500), (1, 901)):
        announce("chunk keys", dtype, bad, D, window, b, at)
        c = Cache([a + n for a, n in zip(news, had)], 2, D, 16, dtype, D)
        key = (int(c.table[b, at // 16]), slice(None), at % 16, 0)
        c.k[key] = bad
        got = mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts), window=window)
        k64 = f64(c.k)
        # a score of -1e30 is one of -inf to the others; where it would be of +inf or NaN the row is left out below
        k64[key] = np.sign(bad) * 1e30 if bad == bad else 0.0
        want, slack, live = ref.chunk_attention(f64(q), k64, f64(c.v), c.table, c.lengths, starts,
                                                np.float64(np.float32(D ** -0.5)), window=window, split=SPLIT[dtype])
        # The slack of such a score is no kernel's: that of a key of score 0 in its place, which at most doubles the
        # sum of the probabilities (the largest is 1), and so at most halves the slack.
        k64[key] = 0.0
        _, slack, _ = ref.chunk_attention(f64(q), k64, f64(c.v), c.table, c.lengths, starts,
                                          np.float64(np.float32(D ** -0.5)), window=window, split=SPLIT[dtype])
        pos = np.concatenate([np.arange(a, a + n) for a, n in zip(had, news)])
        sees = (np.repeat([0, 1], news) == b) & (pos >= at) & ((pos < at + window) if window else True)
        lost = sees[:, None] & ((f64(q)[..., 0] * bad > 0) if bad == bad else np.ones((143, 4), bool))
        mask = torch.from_numpy(lost).cuda()
        assert bool(got[mask].isnan().all())
        within(got[~mask], want[~lost], 2 * slack[~lost])
