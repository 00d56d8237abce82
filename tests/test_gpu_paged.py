"""Attention of single tokens over a paged cache against its 64-bit form: types,
head widths and groups, page sizes, lengths from none to long, windows, sinks,
caps, layouts of the pools, what is never to be read, graphs and streams."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, Cache, f64, i32, within

pytestmark = pytest.mark.gpu

# what a probability loses as the sum of two 16-bit numbers
SPLIT = {torch.bfloat16: 2.0 ** -17, torch.float16: 2.0 ** -22, torch.float32: 0.0}
LENGTHS = [1, 0, 15, 16, 17, 33, 64, 65, 100, 257]


def check(c, q, window=0, softcap=0.0, sinks=None, scale=None, lengths=None, table=None, **kw):
    lengths = c.lengths if lengths is None else lengths
    table = c.table if table is None else table
    s = None if sinks is None else torch.tensor(sinks, dtype=torch.float32).cuda()
    got = mq.paged_attention(q, c.k, c.v, i32(table), i32(lengths), window=window, softcap=softcap, sinks=s,
                             scale=scale, **kw)
    want, slack = ref.attention(f64(q), f64(c.k), f64(c.v), table, lengths, c.D ** -0.5 if scale is None else scale,
                                softcap, window, None if s is None else f64(s), SPLIT[q.dtype])
    within(got, want, slack)
    return got


def query(B, Hq, D, dtype, seed):
    return torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(seed)).to(DTYPES[dtype]).cuda()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 80, 96, 104, 128, 136, 192, 200, 256])
def test_widths(dtype, D):
    announce("paged widths", dtype, D)
    c = Cache(LENGTHS, 2, D, 16, dtype, D)
    check(c, query(len(LENGTHS), 6, D, dtype, D + 1))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (4, 4), (5, 1), (16, 1), (17, 1), (40, 1), (32, 2), (64, 8)])
def test_groups(Hq, Hkv):
    announce("paged groups", Hq, Hkv)
    c = Cache(LENGTHS, Hkv, 64, 16, "bf16", Hq)
    check(c, query(len(LENGTHS), Hq, 64, "bf16", Hq + 1))


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 64, 100, 300])
@pytest.mark.parametrize("window", [0, 1, 20, 128])
def test_pages_and_windows(page, window):
    announce("paged pages", page, window)
    c = Cache(LENGTHS, 2, 128, page, "bf16", page + window)
    check(c, query(len(LENGTHS), 8, 128, "bf16", page), window=window)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("softcap,sinks,window", [(30.0, False, 0), (0.0, True, 0), (5.0, True, 20), (0.0, True, 3)])
def test_cap_and_sinks(dtype, softcap, sinks, window):
    announce("paged cap", dtype, softcap, sinks, window)
    c = Cache(LENGTHS, 2, 96, 16, dtype, 5)
    s = np.linspace(-3, 8, 6) if sinks else None
    check(c, 3 * query(len(LENGTHS), 6, 96, dtype, 6), window, softcap, s)


def test_sinks_of_the_lowest_and_highest_values():
    announce("paged sinks")
    c = Cache([5, 0, 40], 1, 64, 16, "f32", 8)
    q = query(3, 3, 64, "f32", 9)
    check(c, q, sinks=[-np.inf, float(torch.finfo(torch.float32).min), 300.0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["tokens", "joined"])
def test_layouts(dtype, layout):
    announce("paged layouts", dtype, layout)
    c = Cache(LENGTHS, 3, 80, 16, dtype, 11, layout=layout)
    check(c, query(len(LENGTHS), 6, 80, dtype, 12))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_long_and_ragged(dtype):
    announce("paged long", dtype)
    lengths = [5000, 1, 2049, 0, 777, 12000]
    c = Cache(lengths, 2, 128, 16, dtype, 13)
    check(c, query(6, 8, 128, dtype, 14))
    check(c, query(6, 8, 128, dtype, 15), window=1000, sinks=np.zeros(8))


@pytest.mark.parametrize("B", [1, 3, 300])
def test_many_sequences(B):
    announce("paged many", B)
    lengths = [(37 * i * i + 11) % 90 for i in range(B)]
    c = Cache(lengths, 2, 64, 8, "bf16", B)
    check(c, query(B, 4, 64, "bf16", B + 1))


def test_one_long_sequence_of_each_split():
    announce("paged splits")
    for n in (63, 64, 65, 4095, 4096, 4097, 40000):
        c = Cache([n], 1, 64, 32, "bf16", n)
        check(c, query(1, 2, 64, "bf16", n + 1))


@pytest.mark.parametrize("dtype,D,Hq", [("bf16", 80, 5), ("f16", 96, 16), ("bf16", 192, 16), ("f32", 72, 16),
                                        ("f32", 192, 7), ("f32", 256, 16), ("bf16", 256, 40)])
def test_many_joined_parts(dtype, D, Hq):
    """One key head of 40000 keys over more than 16 workgroups, whose results
    are joined in two levels, at widths where a head's columns span waves."""
    announce("paged joined", dtype, D)
    c = Cache([40000], 1, D, 64, dtype, D)
    q = query(1, Hq, D, dtype, D + 1)
    first = check(c, q)
    for _ in range(5):
        assert torch.equal(mq.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lengths)), first)


@pytest.mark.parametrize("length", [2176, 4224, 4352, 8448, 16896])
def test_cut_heads_that_share_a_workgroup(length):
    """Heads of 17, 33, .. workgroups whose last one starts the next cut head."""
    announce("paged shared workgroups", length)
    B = max(2, 40 * 4224 // length // 2)
    c = Cache([length] * B, 2, 64, 16, "bf16", length)
    q = query(B, 2, 64, "bf16", length + 1)
    for _ in range(2):
        check(c, q)


def test_large_scores_and_one_winner():
    announce("paged large")
    c = Cache([200], 1, 64, 16, "f32", 21)
    check(c, 40 * query(1, 4, 64, "f32", 22), scale=1.0)
    c.k[:] = 0  # equal scores: the mean of the values
    got = check(c, query(1, 4, 64, "f32", 23))
    assert torch.equal(got[0, 0], got[0, 3])


def test_scores_of_minus_infinity():
    announce("paged -inf")
    c = Cache([40], 1, 64, 16, "f32", 24)
    page, off = int(c.table[0, 1]), 3
    c.k[page, 0, off] = 0
    c.k[page, 0, off, 0] = float("-inf")
    q = query(1, 2, 64, "f32", 25)
    q[..., 0] = 1.0
    check(c, q)


def test_bad_entries_are_not_followed():
    announce("paged bad entries")
    c = Cache([40, 40, 40], 1, 64, 16, "bf16", 31)
    c.k[:] = torch.randn_like(c.k)
    c.v[:] = torch.randn_like(c.v)
    table = c.table.copy()
    table[1, 1], table[2, 0] = -7, 1 << 30
    q = query(3, 2, 64, "bf16", 32)
    check(c, q, table=table)
    # lengths past the table and below zero
    check(c, q, table=table, lengths=np.array([2 ** 31 - 1, -5, 48], np.int32))


def test_query_and_out_of_any_strides():
    announce("paged strides")
    c = Cache([70, 3], 2, 64, 16, "bf16", 41)
    q = query(2, 4, 64, "bf16", 42)
    want = mq.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lengths))
    wide = torch.randn(2, 9, 130, device="cuda").to(torch.bfloat16)
    wide[:, 1:5, 3:67] = q
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (wide[:, 1:5, 3:67], turned):
        assert torch.equal(mq.paged_attention(x, c.k, c.v, i32(c.table), i32(c.lengths)), want)
    out = torch.zeros(2, 64, 4, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    assert mq.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lengths), out=out) is out
    assert torch.equal(out, want)
    table = torch.zeros(2, 20, dtype=torch.int32, device="cuda")
    table[:, 7:7 + c.width] = i32(c.table)
    assert torch.equal(mq.paged_attention(q, c.k, c.v, table[:, 7:7 + c.width], i32(c.lengths)), want)


def test_offsets_past_32_bits():
    announce("paged far pages")
    D, page, far = 64, 16, (1 << 32) // (64 * 16) + 40  # page `far` begins past 2^32 elements
    k, v = (torch.empty(far + 2, 1, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    small = Cache([30], 1, D, page, "bf16", 51)
    for j in range(2):
        k[far + j] = small.k[int(small.table[0, j])]
        v[far + j] = small.v[int(small.table[0, j])]
    q = query(1, 2, D, "bf16", 52)
    got = mq.paged_attention(q, k, v, i32([[far, far + 1]]), i32([30]))
    assert torch.equal(got, mq.paged_attention(q, small.k, small.v, i32(small.table), i32([30])))


def test_no_sequences_and_repeatable():
    c = Cache([5000, 20], 2, 64, 16, "bf16", 61)
    q = query(2, 4, 64, "bf16", 62)
    none = mq.paged_attention(q[:0], c.k, c.v, i32(c.table)[:0], i32(c.lengths)[:0])
    assert none.shape == (0, 4, 64)
    first = mq.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lengths))
    for _ in range(3):
        assert torch.equal(mq.paged_attention(q, c.k, c.v, i32(c.table), i32(c.lengths)), first)


def test_graph_and_another_stream():
    announce("paged graph")
    lengths = [700, 9000, 1]
    c = Cache(lengths, 2, 64, 16, "bf16", 71)
    q, table, n = query(3, 8, 64, "bf16", 72), i32(c.table), i32(lengths)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager = mq.paged_attention(q, c.k, c.v, table, n)
    s.synchronize()
    assert torch.equal(eager, mq.paged_attention(q, c.k, c.v, table, n))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        mq.paged_attention(q, c.k, c.v, table, n, out=out)
    for lens in ([700, 9000, 1], [3, 8192, 0], [0, 0, 0], [640, 20, 1]):
        n.copy_(i32(lens))
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want, slack = ref.attention(f64(q), f64(c.k), f64(c.v), c.table, lens, 64 ** -0.5, split=SPLIT[q.dtype])
        within(out, want, slack, lens)


def test_the_ctypes_path_gives_the_same(monkeypatch):
    from mlxcel_amd import ops

    c = Cache([33, 5], 2, 64, 16, "f16", 81)
    q, args = query(2, 4, 64, "f16", 82), (i32(c.table), i32(c.lengths))
    want = mq.paged_attention(q, c.k, c.v, *args, window=9, softcap=20.0)
    monkeypatch.setattr(ops, "_native", ops._ctypes_only)
    assert torch.equal(mq.paged_attention(q, c.k, c.v, *args, window=9, softcap=20.0), want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_probabilities_keep_32_bits(dtype):
    """Sequences of three keys with scores 0, 0 and x < 0, values -a, -b and 1, where a is
    p = exp(x) in the pool's type and b what is left of it: (p - a - b) / (2 + p), what a
    probability held in two numbers of bfloat16 has lost.  Of p in 32 bits 3 |x| u
    are the score's roundings, 2 u the exponential's, 8 u the sums', u = 2^-24."""
    announce("paged probabilities", dtype)
    t, n, u = DTYPES[dtype], 128, 2.0 ** -24
    x = -torch.arange(1, n + 1, dtype=torch.float64) / 256
    p = x.exp()
    a = p.to(t)
    b = (p - a.double()).to(t)
    want = ((p - a.double() - b.double()) / (2 + p))[:, None].numpy()
    slack = ((3 * x.abs() + 10) * u * p / (2 + p))[:, None].numpy()
    if dtype == "bf16":
        assert (np.abs(want) > 2 * slack).sum() > n / 4  # zeros would not do
    k, v = torch.zeros(n, 1, 3, 8, dtype=t), torch.zeros(n, 1, 3, 8, dtype=t)
    k[:, 0, 2, 0] = x.to(t)
    v[:, 0] = torch.stack([-a, -b, torch.ones_like(a)], 1)[:, :, None]
    q = torch.zeros(n, 1, 8, dtype=t)
    q[..., 0] = 1
    got = mq.paged_attention(q.cuda(), k.cuda(), v.cuda(), i32(np.arange(n)[:, None]), i32([3] * n), scale=1.0)
    within(got[:, 0], np.broadcast_to(want, (n, 8)), slack)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 40, 700, 20000])
def test_scores_that_are_all_minus_infinity(dtype, n):
    """NaN as softmax gives, unless a sink joins: then zeros.  Where some scores are
    -inf, the keys that are left alone."""
    announce("paged all -inf", dtype, n)
    c = Cache([n], 1, 64, 16, dtype, n)
    q = query(1, 3, 64, dtype, n + 1)
    q[..., 0] = 1.0
    ok = torch.isfinite(c.k[:, :, :, 0])
    c.k[..., 0] = torch.where(ok, -float("inf"), c.k[..., 0])
    args = (q, c.k, c.v, i32(c.table), i32(c.lengths))
    sinks = torch.tensor([0.0, -float("inf"), -3e38], device="cuda")
    assert torch.isnan(mq.paged_attention(*args)).all()
    got = mq.paged_attention(*args, sinks=sinks)
    assert not got[0, [0, 2]].any() and torch.isnan(got[0, 1]).all()
    few = Cache([n], 1, 64, 16, dtype, n + 2)
    at = np.arange(n)
    pages, off = few.table[0, at // 16], at % 16
    gone = np.random.default_rng(n).random(n) < 0.5
    gone[n // 2] = False
    few.k[pages[gone], 0, off[gone], 0] = -float("inf")
    k, v = (t[pages[~gone], 0, off[~gone]][None, None] for t in (few.k, few.v))
    want, slack = ref.attention(f64(q), f64(k), f64(v), np.zeros((1, 1), np.int32), [k.shape[2]], 0.125)
    within(mq.paged_attention(q, few.k, few.v, i32(few.table), i32(few.lengths)), want, slack + n * ref.U * np.abs(want))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [40, 20000])
def test_largest_finite_sinks(dtype, n):
    announce("paged largest sinks", dtype, n)
    top = float(torch.finfo(torch.float32).max)
    c = Cache([n], 1, 64, 16, dtype, n)
    got = check(c, query(1, 6, 64, dtype, n + 1), sinks=[top, 2.5e38, -top, -2.5e38, np.inf, -np.inf])
    assert not got[0, :2].any() and torch.isnan(got[0, 4]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [40, 20000])
def test_infinite_values(dtype, n):
    """32-bit pools add them up; in 16-bit ones an infinite value makes its column
    infinite or NaN.  Other columns and the sequence beside it are left alone."""
    announce("paged infinite values", dtype, n)
    inf = float("inf")
    c = Cache([n, 33], 1, 64, 16, dtype, n)
    q = query(2, 3, 64, dtype, n + 1)
    args = (q, c.k, c.v, i32(c.table), i32(c.lengths))
    want = mq.paged_attention(*args)
    at = lambda t: (int(c.table[0, t // 16]), 0, t % 16)
    for t, column, value in ((0, 3, inf), (n - 1, 5, -inf), (0, 7, inf), (n - 1, 7, -inf), (n // 2, 9, float("nan"))):
        c.v[at(t)][column] = value
    got = mq.paged_attention(*args)
    bad = [3, 5, 7, 9]
    rest = [d for d in range(64) if d not in bad]
    assert torch.equal(got[1], want[1]) and torch.equal(got[0][:, rest], want[0][:, rest])
    assert torch.isnan(got[0][:, [7, 9]]).all()
    if dtype == "f32":
        assert (got[0][:, 3] == inf).all() and (got[0][:, 5] == -inf).all()
    else:
        assert not torch.isfinite(got[0][:, [3, 5]]).any()


def test_copies_take_their_own_size():
    announce("paged staging size")
    B, H, mib = 64, 64, 1 << 20
    c = Cache([5] * B, 1, 256, 16, "f32", 91)
    q, args = query(B, H, 256, "f32", 92), (c.k, c.v, i32(c.table), i32(c.lengths))  # 4 MiB
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    out = torch.empty(B, 256, H, device="cuda").transpose(1, 2)
    want = mq.paged_attention(q, *args)
    torch.cuda.synchronize()
    mq.clear_cache()
    mq.paged_attention(q, *args)
    held = mq.get_cache_memory()
    assert torch.equal(mq.paged_attention(turned, *args), want)
    assert mq.get_cache_memory() == held + 4 * mib
    assert torch.equal(mq.paged_attention(turned, *args, out=out), want)
    assert mq.get_cache_memory() == held + (4 + 8) * mib  # the first buffer is kept until clear_cache


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window", [0, 30000])
def test_more_than_the_last_cache_holds(dtype, window):
    """Past 128 MiB of keys and values they are read past it."""
    announce("paged past the cache", dtype, window)
    lengths = [40000, 1, 0, 25001]
    c = Cache(lengths, 8, 128, 64, dtype, 95)
    q = query(4, 16, 128, dtype, 96)
    seen = sum(min(n, window or n) for n in lengths)
    assert seen * 2 * 8 * 128 * q.element_size() > 128 << 20
    got = mq.paged_attention(q, c.k, c.v, i32(c.table), i32(lengths), window=window)
    for h in range(8):  # 64-bit keys and values of one head at a time
        mine = slice(2 * h, 2 * h + 2)
        want, slack = ref.attention(f64(q[:, mine]), f64(c.k[:, h:h + 1]), f64(c.v[:, h:h + 1]), c.table, lengths,
                                    128 ** -0.5, 0.0, window)
        within(got[:, mine], want, slack, h)


MIXED = [0, 1, 100, 200, 300, 400, 500, 513, 2000, 3000]


def mixed(B, seed, most=9000):
    g = np.random.default_rng(seed)
    lengths = g.choice(MIXED, B)
    lengths[[0, B // 2, B - 1]] = most, 0, most - 1
    return lengths.astype(np.int32)


@pytest.mark.parametrize("B", [63, 64, 65, 200, 256, 257, 600])
@pytest.mark.parametrize("window,sinks", [(0, False), (300, True), (2500, False)])
def test_many_sequences_with_cut_heads(B, window, sinks):
    """Sequences without keys, heads of one to four steps and cut ones, on both
    sides of 64 sequences and of one a thread."""
    announce("paged many cut", B, window, sinks)
    c = Cache(mixed(B, B + window).tolist(), 2, 64, 16, "bf16", B)
    check(c, query(B, 4, 64, "bf16", B + 1), window, 0.0, np.linspace(-2, 4, 4) if sinks else None)


@pytest.mark.parametrize("B", [64, 65, 300])
def test_graph_of_many_sequences(B):
    announce("paged many graph", B)
    most = mixed(B, 1, 9000)
    first = np.maximum(most, 600)
    c = Cache(first.tolist(), 2, 64, 16, "bf16", B)
    for t in (c.k, c.v):  # lengths are changed within the rows' pages
        t[torch.isnan(t)] = 0.5
    q, table, n = query(B, 4, 64, "bf16", B + 1), i32(c.table), i32(first)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        mq.workspace_reserve(32 << 20)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        mq.paged_attention(q, c.k, c.v, table, n, out=out)
    for rep, lens in enumerate((first, np.minimum(first, 130), np.where(np.arange(B) % 7 == 3, first, 0), first * 0, most)):
        n.copy_(i32(lens))
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want, slack = ref.attention(f64(q), f64(c.k), f64(c.v), c.table, lens, 64 ** -0.5)
        within(out, want, slack, rep)
