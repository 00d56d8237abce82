"""Attention of several new tokens per sequence over the paged cache against
the 64-bit form, one token at a time.

Tolerance: oracle.serving.attention's slack (each score's rounding and the
sums'), SPLIT's relative loss of a probability, and the rounding to the type.
Slots of the pools that no sequence holds are NaN: reading one shows."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, Cache, f64, i32, within

pytestmark = pytest.mark.gpu

# 16-bit products take a probability as the sum of two numbers: the second leaves
# out half a step of what the first left, 2^-8 * 2^-9 and 2^-11 * 2^-12 (float16
# also 2^-39 of the largest, which is below that for n < 2^16 keys).
SPLIT = {"bf16": 2.0 ** -17, "f16": 2.0 ** -23, "f32": 0.0}


def starts_of(news):
    return np.concatenate([[0], np.cumsum(news)]).astype(np.int32)


def queries(T, Hq, D, dtype, seed, by=1.0):
    g = torch.Generator().manual_seed(seed)
    return (by * torch.randn(T, Hq, D, generator=g)).to(DTYPES[dtype]).cuda()


def check(c, q, starts, dtype, got=None, lengths=None, **kw):
    lengths = c.lengths if lengths is None else lengths
    if got is None:
        s = kw.get("sinks")
        got = mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(lengths), i32(starts),
                                       **{**kw, "sinks": None if s is None else torch.from_numpy(s).cuda()})
    scale = kw.get("scale")
    scale = np.float64(np.float32(q.shape[-1] ** -0.5 if scale is None else scale))
    want, slack, live = ref.chunk_attention(f64(q), f64(c.k), f64(c.v), c.table, lengths, starts, scale,
                                            kw.get("softcap", 0.0), kw.get("window", 0), kw.get("sinks"), SPLIT[dtype])
    within(got[torch.from_numpy(live).cuda()], want[live], slack[live])
    return got


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 64, 16), (3, 3, 128, 16), (5, 1, 80, 24), (4, 2, 96, 8), (2, 1, 192, 1),
                                           (4, 4, 256, 32), (16, 1, 8, 5), (40, 2, 72, 64)])
def test_heads_widths_pages(dtype, Hq, Hkv, D, page):
    announce("chunk widths", dtype, Hq, Hkv, D, page)
    news, had = [1, 7, 40, 0, 33], [0, 30, 11, 50, 64]
    c = Cache([a + b for a, b in zip(news, had)], Hkv, D, page, dtype, D)
    check(c, queries(sum(news), Hq, D, dtype, Hq), starts_of(news), dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("new,had", [(1, 0), (2, 0), (1, 1), (31, 0), (32, 0), (33, 0), (64, 64), (65, 63), (127, 1), (128, 0),
                                     (129, 500), (1, 700), (5, 1021), (300, 0), (257, 255)])
def test_lengths(dtype, new, had):
    announce("chunk lengths", dtype, new, had)
    c = Cache([new + had], 2, 64, 16, dtype, new + had)
    check(c, queries(new, 6, 64, dtype, new), starts_of([new]), dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 100, 128, 1000])
def test_windows(dtype, window):
    announce("chunk windows", dtype, window)
    news, had = [70, 3, 1], [0, 150, 333]
    c = Cache([a + b for a, b in zip(news, had)], 1, 64, 16, dtype, window)
    check(c, queries(sum(news), 4, 64, dtype, window), starts_of(news), dtype, window=window)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(scale=0.0), dict(scale=-0.3), dict(scale=1.5),
                                dict(sinks=True), dict(sinks=True, window=20, softcap=5.0), dict(scale=-0.2, softcap=3.0)])
def test_scores(dtype, kw):
    announce("chunk scores", dtype, kw)
    news, had = [37, 2], [20, 90]
    c = Cache([a + b for a, b in zip(news, had)], 2, 64, 16, dtype, 3)
    kw = dict(kw)
    if kw.get("sinks"):
        kw["sinks"] = np.random.default_rng(2).normal(size=6).astype(np.float32) * 3
    check(c, queries(39, 6, 64, dtype, 5), starts_of(news), dtype, **kw)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("layout", ["pages", "tokens", "both"])
def test_layouts(dtype, layout):
    announce("chunk layouts", dtype, layout)
    news, had = [20, 1, 50], [3, 70, 0]
    c = Cache([a + b for a, b in zip(news, had)], 3, 40, 12, dtype, 4, layout=layout)
    check(c, queries(71, 6, 40, dtype, 6), starts_of(news), dtype)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_strided_q_and_out(dtype):
    announce("chunk strides", dtype)
    news, had = [9, 30], [5, 2]
    c = Cache([a + b for a, b in zip(news, had)], 2, 64, 16, dtype, 4)
    starts = starts_of(news)
    fused = queries(39, 10, 64, dtype, 1)
    q = fused[:, 1:7]
    out = torch.zeros(6, 39, 64, dtype=q.dtype, device="cuda").transpose(0, 1)
    assert mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts), out=out) is out
    check(c, q, starts, dtype, got=out)
    odd = torch.cat([fused.reshape(39, -1), fused[:, :1, :3].reshape(39, -1)], 1)[:, 1:1 + 6 * 64].view(39, 6, 64)
    check(c, odd, starts, dtype)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert turned.stride(2) != 1
    check(c, turned, starts, dtype)


@pytest.mark.parametrize("strided", [False, True])
def test_rows_of_no_sequence_stay(strided):
    announce("chunk padding", strided)
    c = Cache([20, 9], 2, 64, 16, "bf16", 1)
    q = queries(40, 4, 64, "bf16", 2)
    starts = np.int32([3, 10, 19])
    out = torch.full((4, 40, 64) if strided else (40, 4, 64), 7.0, dtype=q.dtype, device="cuda")
    out = out.transpose(0, 1) if strided else out
    mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32(starts), out=out)
    check(c, q, starts, "bf16", got=out)
    assert bool((out[:3] == 7).all()) and bool((out[19:] == 7).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_more_rows_than_tokens(dtype):
    """Rows before a sequence's first token give zeros, as do all of a sequence of length 0 or less; sinks too."""
    announce("chunk short", dtype)
    c = Cache([4, 0, 0, 3], 1, 64, 16, dtype, 1)
    starts, lengths = np.int32([0, 10, 15, 17, 20]), np.int32([4, 0, -5, 3])
    q = queries(20, 2, 64, dtype, 3)
    sinks = np.float32([0.5, -1])
    for s in (None, sinks):
        got = check(c, q, starts, dtype, lengths=lengths, sinks=s)
        assert bool((got[:6] == 0).all()) and bool((got[10:17] == 0).all())


def test_lengths_past_the_table():
    announce("chunk capacity")
    c = Cache([32], 1, 64, 16, "bf16", 1)
    check(c, queries(5, 2, 64, "bf16", 3), np.int32([0, 5]), "bf16", lengths=np.int32([1000]))


def test_pages_out_of_range_are_clamped():
    announce("chunk clamped pages")
    c = Cache([64], 2, 64, 16, "f32", 1, spare=0)
    q = queries(10, 2, 64, "f32", 3)
    c.table[0, 1], c.table[0, 2] = -7, 2 ** 31 - 1
    check(c, q, np.int32([0, 10]), "f32")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_later_tokens_do_not_reach_earlier_ones(dtype, bad):
    """Keys and values that are not finite change the tokens that see them and no other."""
    announce("chunk masked values", dtype, bad)
    n, had, at = 100, 30, 95
    c = Cache([n + had], 1, 64, 16, dtype, 1)
    q = queries(n, 4, 64, dtype, 3)
    args = (i32(c.table), i32(c.lengths), i32([0, n]))
    want = mq.paged_attention_chunk(q, c.k, c.v, *args)
    for pool in (c.k, c.v):
        p = int(c.table[0, at // 16])
        was = pool[p, 0, at % 16].clone()
        pool[p, 0, at % 16] = bad
        got = mq.paged_attention_chunk(q, c.k, c.v, *args)
        assert torch.equal(got[:at - had], want[:at - had])
        if pool is c.v:
            assert not bool(torch.isfinite(got[at - had:]).any())
        got = mq.paged_attention_chunk(q, c.k, c.v, *args, window=10)
        seen = mq.paged_attention_chunk(q, c.k, c.v, *args, window=10)
        assert bool(torch.isfinite(got[:at - had]).all()) and bool(torch.isfinite(got[at - had + 10:]).all())
        pool[p, 0, at % 16] = was


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_scores_that_are_all_minus_infinity(dtype):
    announce("chunk -inf scores", dtype)
    c = Cache([40], 1, 64, 16, dtype, 1)
    q = queries(8, 2, 64, dtype, 3)
    q[3, 1, 5] = float("inf")
    for p in c.table[0]:
        c.k[p, 0, :, 5] = torch.where(c.k[p, 0, :, 5].isnan(), c.k[p, 0, :, 5], torch.tensor(-1.0, dtype=c.k.dtype, device="cuda"))
    got = mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32([0, 8]))
    nan = got.isnan().all(-1)
    assert bool(nan[3, 1]) and int(nan.sum()) == 1 and int(got.isnan().any(-1).sum()) == 1
    sinks = torch.tensor([0.0, 0.0], device="cuda")
    got = mq.paged_attention_chunk(q, c.k, c.v, i32(c.table), i32(c.lengths), i32([0, 8]), sinks=sinks)
    assert bool((got[3, 1] == 0).all()) and bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_peaked_and_growing_scores(dtype):
    """Scores of hundreds whose maximum grows along the keys; probabilities that underflow."""
    announce("chunk peaked", dtype)
    c = Cache([300], 1, 64, 16, dtype, 1)
    ramp = torch.zeros(c.pages, device="cuda")
    for j, p in enumerate(c.table[0]):
        ramp[p] = 0.2 * j
    c.k = (c.k.float() * (1 + ramp[:, None, None, None])).to(c.k.dtype)
    check(c, queries(150, 2, 64, dtype, 3, by=8.0), np.int32([0, 150]), dtype)


@pytest.mark.parametrize("B", [1, 63, 64, 65, 300])
def test_many_sequences(B):
    """Ragged batches: single tokens, short prompts, nothing new, empty ones."""
    announce("chunk batch", B)
    r = np.random.default_rng(B)
    news = np.where(r.random(B) < 0.5, 1, r.integers(0, 20, B))
    had = np.where(r.random(B) < 0.2, 0, r.integers(0, 200, B))
    c = Cache((news + had).tolist(), 2, 64, 16, "bf16", B)
    check(c, queries(int(news.sum()), 4, 64, "bf16", B), starts_of(news), "bf16")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (130, 1), (256, 2), (48, 16)])
def test_many_heads_over_long_caches(dtype, Hq, Hkv):
    """Heads of one key head past a tile, and caches that several workgroups share."""
    announce("chunk long", dtype, Hq, Hkv)
    news, had = [3, 1], [3000, 1700]
    c = Cache([a + b for a, b in zip(news, had)], Hkv, 64, 16, dtype, 2)
    check(c, queries(4, Hq, 64, dtype, 3), starts_of(news), dtype)


def test_a_prompt_in_parts():
    """A prompt in one call, in parts, and its last token with paged_attention: all within the same slack."""
    announce("chunk parts")
    c = Cache([500], 2, 128, 16, "bf16", 7)
    q = queries(500, 8, 128, "bf16", 8)
    check(c, q, np.int32([0, 500]), "bf16")
    for cut in ((0, 1, 300, 500), (0, 128, 256, 384, 500), (0, 499, 500)):
        for a, b in zip(cut[:-1], cut[1:]):
            check(c, q[a:b], np.int32([0, b - a]), "bf16", lengths=np.int32([b]))
    one = mq.paged_attention(q[-1:], c.k, c.v, i32(c.table), i32([500]))
    check(c, q[-1:], np.int32([0, 1]), "bf16", got=one)


def test_the_same_bits_every_time():
    announce("chunk again")
    c = Cache([9000, 50], 1, 64, 16, "bf16", 7)
    q = queries(60, 8, 64, "bf16", 8)
    args = (q, c.k, c.v, i32(c.table), i32(c.lengths), i32([0, 30, 60]))
    first = mq.paged_attention_chunk(*args)
    for _ in range(20):
        assert torch.equal(mq.paged_attention_chunk(*args), first)


def test_two_streams_at_once():
    announce("chunk streams")
    cs = [Cache([3000 + 500 * i, 40], 2, 64, 16, "bf16", i) for i in range(2)]
    qs = [queries(50, 4, 64, "bf16", i) for i in range(2)]
    args = [(q, c.k, c.v, i32(c.table), i32(c.lengths), i32([0, 25, 50])) for q, c in zip(qs, cs)]
    want = [mq.paged_attention_chunk(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(mq.paged_attention_chunk(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_graph_of_growing_sequences():
    """Two graphs captured on one stream (they share its workspaces), replayed in turn while the lengths grow."""
    announce("chunk graph")
    c = Cache([2000, 700], 2, 64, 16, "bf16", 3)
    q = queries(64, 4, 64, "bf16", 4)
    table, lengths, starts = i32(c.table), i32([100, 50]), i32([0, 32, 64])
    graphs, outs, side = [], [], torch.cuda.Stream()
    for window in (0, 40):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # its workspaces, before the capture
            mq.paged_attention_chunk(q, c.k, c.v, table, lengths, starts, window=window)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(mq.paged_attention_chunk(q, c.k, c.v, table, lengths, starts, window=window))
        graphs.append(g)
    for step, (a, b, cut) in enumerate([(64, 32, 32), (1999, 650, 1), (2000, 64, 60), (500, 700, 0)]):
        lengths.copy_(i32([a, b]))
        starts.copy_(i32([0, cut, 64]))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        eager = mq.paged_attention_chunk(q, c.k, c.v, table, lengths, starts)
        assert torch.equal(outs[0], eager)
        check(c, q, np.int32([0, cut, 64]), "bf16", got=outs[0], lengths=np.int32([a, b]))
        check(c, q, np.int32([0, cut, 64]), "bf16", got=outs[1], lengths=np.int32([a, b]), window=40)


def test_pools_past_4_gib():
    announce("chunk far pages")
    pages = (5 << 30) // (2 * 64 * 128 * 2)
    k = torch.zeros(pages, 2, 64, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    near = Cache([200], 2, 128, 64, "bf16", 5)
    table = near.table.copy()
    for j in range(4):
        k[pages - 1 - j], v[pages - 1 - j] = near.k[int(table[0, j])], near.v[int(table[0, j])]
        table[0, j] = pages - 1 - j
    q = queries(40, 4, 128, "bf16", 6)
    got = mq.paged_attention_chunk(q, k, v, i32(table), i32([200]), i32([0, 40]))
    want = mq.paged_attention_chunk(q, near.k, near.v, i32(near.table), i32([200]), i32([0, 40]))
    assert torch.equal(got, want)
