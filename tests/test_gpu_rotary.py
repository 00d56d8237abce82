"""Position rotations against the 64-bit form: layouts, types, parts of a head,
far and negative positions, strides, in place, on the way into the cache.

Tolerance: oracle.serving.rotary's slack and the rounding to the type."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, Cache, f64, i32, within

pytestmark = pytest.mark.gpu


def heads(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(DTYPES[dtype]).cuda()


def freq(n, base=10000.0):
    return (base ** (-np.arange(n) / max(n, 1))).astype(np.float32)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,n", [
    (1, 1, 2, 1), (1, 32, 128, 64), (3, 5, 80, 10), (17, 3, 96, 32), (5, 2, 7, 3), (2, 40, 256, 128), (4, 1, 64, 0),
    (300, 8, 72, 9), (1, 300, 64, 32), (2, 2, 4096, 2048), (3, 1, 33, 16),
])
def test_rotary(dtype, interleaved, T, H, D, n):
    announce("rotary", dtype, interleaved, T, H, D, n)
    x = heads((T, H, D), dtype, T + D)
    pos = np.random.default_rng(D).integers(0, 5000, T)
    y = mq.rotary(x, i32(pos), torch.from_numpy(freq(n)).cuda(), interleaved=interleaved, factor=1.25)
    want, slack = ref.rotary(f64(x), pos, freq(n), interleaved, np.float64(np.float32(1.25)))
    within(y, want, slack)
    assert torch.equal(y[..., 2 * n:], x[..., 2 * n:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pos", [[0, 1, -1], [131071, 1000003, -1000003], [2 ** 20 - 1, 2 ** 20, -2 ** 20]])
def test_far_and_negative_positions(interleaved, pos):
    announce("rotary far", interleaved, pos)
    x = heads((3, 2, 64), "f32", 5)
    y = mq.rotary(x, i32(pos), torch.from_numpy(freq(32)).cuda(), interleaved=interleaved)
    within(y, *ref.rotary(f64(x), np.array(pos), freq(32), interleaved))


def test_quarter_turns():
    """Angles at and next to multiples of an eighth of a turn, where the series change places."""
    announce("rotary quarters")
    pos = np.arange(-40, 41)
    f = np.concatenate([np.float32([np.pi / 4, np.pi / 2, np.pi]), np.nextafter(np.float32([np.pi / 4, np.pi / 2]), 9, dtype=np.float32)])
    x = heads((len(pos), 1, 10), "f32", 6)
    y = mq.rotary(x, i32(pos), torch.from_numpy(f).cuda())
    within(y, *ref.rotary(f64(x), pos, f))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("interleaved", [False, True])
def test_views_and_in_place(dtype, interleaved):
    announce("rotary views", dtype, interleaved)
    inv, pos = torch.from_numpy(freq(16)).cuda(), np.arange(7) * 31
    fused = heads((7, 2 + 4 * 48 + 1), dtype, 9)
    x = fused[:, 1:1 + 4 * 48].view(7, 4, 48)  # rows of odd stride and offset
    want, slack = ref.rotary(f64(x), pos, freq(16), interleaved)
    within(mq.rotary(x, i32(pos), inv, interleaved=interleaved), want, slack, "view")
    out = torch.zeros(4, 7, 48, dtype=x.dtype, device="cuda").transpose(0, 1)
    assert mq.rotary(x, i32(pos), inv, interleaved=interleaved, out=out) is out
    within(out, want, slack, "out of other strides")
    last = x.transpose(1, 2).contiguous().transpose(1, 2)  # the last axis strided
    assert last.stride(2) != 1
    out = torch.zeros_like(last)
    mq.rotary(last, i32(pos), inv, interleaved=interleaved, out=out)
    within(out, want, slack, "last axis strided")
    before = fused.clone()
    mq.rotary(x, i32(pos), inv, interleaved=interleaved, out=x)
    within(x, want, slack, "in place")
    assert torch.equal(fused[:, 0], before[:, 0]) and torch.equal(fused[:, 1 + 4 * 48:], before[:, 1 + 4 * 48:])
    one = heads((1, 4, 48), dtype, 3).expand(7, 4, 48)  # one row for all tokens
    within(mq.rotary(one, i32(pos), inv, interleaved=interleaved), *ref.rotary(f64(one), pos, freq(16), interleaved))


def test_empty():
    announce("rotary empty")
    inv = torch.ones(4, device="cuda")
    for shape in ((0, 2, 8), (3, 0, 8)):
        assert mq.rotary(torch.zeros(shape, device="cuda"), i32(np.zeros(shape[0])), inv).shape == shape


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(interleaved):
    """d(g . rotary(x)) / dx is rotary of g at the negated positions: against the 64-bit form's differences."""
    announce("rotary gradient", interleaved)
    pos, f = np.array([3, 1000, 70000]), freq(6)
    x, g = heads((3, 2, 14), "f32", 1), heads((3, 2, 14), "f32", 2)
    got = mq.rotary(g, -i32(pos), torch.from_numpy(f).cuda(), interleaved=interleaved, factor=1.5)
    want, slack = ref.rotary(f64(g), -pos, f, interleaved, 1.5)
    within(got, want, slack)
    x0, d = f64(x), np.zeros((3, 2, 14))
    for i in np.ndindex(d.shape):
        e = np.zeros(d.shape)
        e[i] = 0.5  # the rotation is linear: any step is exact up to rounding
        d[i] = (f64(g) * (ref.rotary(x0 + e, pos, f, interleaved, 1.5)[0] - ref.rotary(x0 - e, pos, f, interleaved, 1.5)[0])).sum()
    d[..., 12:] = f64(g)[..., 12:]
    np.testing.assert_allclose(want, d, atol=1e-11)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("layout", ["pages", "tokens", "padded"])
@pytest.mark.parametrize("interleaved,Hq,Hkv,D,n,page", [(False, 8, 2, 64, 32, 16), (True, 5, 5, 40, 10, 3), (False, 1, 1, 20, 5, 1),
                                                         (True, 32, 8, 128, 64, 24)])
def test_rotary_append(dtype, layout, interleaved, Hq, Hkv, D, n, page):
    announce("rotary append", dtype, layout, interleaved, Hq, Hkv, D, n, page)
    lengths = [7, 0, 33, 1]
    c = Cache(lengths, Hkv, D, page, dtype, D)
    if layout == "tokens":
        c.k, c.v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k, c.v))
    elif layout == "padded":
        pad = torch.zeros(*c.k.shape[:3], 2, dtype=c.k.dtype, device="cuda")
        c.k, c.v = (torch.cat([t, pad], -1)[..., :D] for t in (c.k, c.v))
    # tokens of every row, and some that have no place: row, position, page, length
    rows = np.array([0, 0, 2, 2, 3, 0, -1, 4, 2, 2, 1, 2, 0])
    pos = np.array([6, 0, 32, 15, 0, 3, 0, 0, -1, 10 ** 6, 0, 33, 7])
    table = c.table.copy()
    T = len(rows)
    q, k, v = heads((T, Hq, D), dtype, 1), heads((T, Hkv, D), dtype, 2), heads((T, Hkv, D), dtype, 3)
    inv = torch.from_numpy(freq(n)).cuda()
    k0, v0 = c.k.clone(), c.v.clone()
    got = mq.rotary_append(q, k, v, c.k, c.v, i32(table), i32(pos), i32(rows), inv, lengths=i32(c.lengths),
                           interleaved=interleaved, factor=0.75)
    within(got, *ref.rotary(f64(q), pos, freq(n), interleaved, 0.75), "q")
    turned, slack = ref.rotary(f64(k), pos, freq(n), interleaved, 0.75)
    wrote = torch.zeros(c.k.shape[:3], dtype=torch.bool, device="cuda")
    for t in range(6):
        at = (int(table[rows[t], pos[t] // page]), slice(None), int(pos[t] % page))
        within(c.k[at], turned[t], slack[t], ("k", t))
        assert torch.equal(c.v[at], v[t])
        wrote[at] = True
    for a, b in ((c.k, k0), (c.v, v0)):
        same = (a == b) | (a.isnan() & b.isnan())
        assert bool(same[~wrote].all())
    # the same as rotary and cache_append
    mq.cache_append(mq.rotary(k, i32(pos), inv, interleaved=interleaved, factor=0.75), v, k0, v0, i32(table), i32(pos),
                    i32(rows), lengths=i32(c.lengths))
    for a, b in ((c.k, k0), (c.v, v0)):
        assert bool(((a == b) | (a.isnan() & b.isnan())).all())


def test_append_pages_out_of_range():
    announce("rotary append pages")
    c = Cache([16], 2, 16, 8, "bf16", 0)
    k0 = c.k.clone()
    k = heads((3, 2, 16), "bf16", 1)
    inv = torch.from_numpy(freq(8)).cuda()
    table = np.array([[-1, c.pages, 2 ** 31 - 1]], np.int32)
    mq.rotary_append(k, k, k, c.k, c.v, i32(table), i32([0, 8, 16]), i32([0, 0, 0]), inv)
    assert bool(((c.k == k0) | (c.k.isnan() & k0.isnan())).all())
    # a table without columns takes no token, the queries are rotated
    got = mq.rotary_append(k, k, k, c.k, c.v, i32(np.zeros((1, 0))), i32([0, 8, 16]), i32([0, 0, 0]), inv)
    within(got, *ref.rotary(f64(k), np.array([0, 8, 16]), freq(8)))
    assert bool(((c.k == k0) | (c.k.isnan() & k0.isnan())).all())


def test_append_in_place_and_of_a_fused_projection():
    announce("rotary append fused")
    c = Cache([5, 40], 2, 32, 16, "f16", 3)
    fused = heads((4, (6 + 4) * 32), "f16", 4)
    q, k, v = (t.view(4, -1, 32) for t in fused.split((6 * 32, 64, 64), 1))
    pos, rows = np.array([4, 39, 38, 0]), np.array([0, 1, 1, 0])
    want, slack = ref.rotary(f64(q), pos, freq(16))
    kv = fused[:, 6 * 32:].clone()
    inv = torch.from_numpy(freq(16)).cuda()
    assert mq.rotary_append(q, k, v, c.k, c.v, i32(c.table), i32(pos), i32(rows), inv, out=q) is q
    within(q, want, slack)
    assert torch.equal(fused[:, 6 * 32:], kv)
    strided = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]  # the last axis strided
    before = c.k.clone(), c.v.clone()
    mq.rotary_append(q, *strided, c.k, c.v, i32(c.table), i32(pos), i32(rows), inv)
    for a, b in zip((c.k, c.v), before):
        assert bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("past", [False, True])
def test_offsets_past_32_bits(past):
    """Pages whose elements lie past 2^32 bytes of the pool."""
    announce("rotary append far pages", past)
    pages = (5 << 30) // (2 * 64 * 128 * 2)
    pool = torch.zeros(pages, 2, 64, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(pool)
    k = heads((2, 2, 128), "bf16", 1)
    at = pages - 1 if past else 0
    mq.rotary_append(k, k, k, pool, v, i32([[at]]), i32([0, 63]), i32([0, 0]), torch.from_numpy(freq(64)).cuda())
    assert torch.equal(v[at, :, 0], k[0]) and torch.equal(v[at, :, 63], k[1])
    within(pool[at, :, 63], *(t[1] for t in ref.rotary(f64(k), np.array([0, 63]), freq(64))))


def test_graph_and_streams():
    """A captured call replayed on new positions, eager calls on another stream between the replays."""
    announce("rotary graph")
    inv = torch.from_numpy(freq(32)).cuda()
    x, pos = heads((9, 4, 64), "bf16", 1), i32(np.arange(9))
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mq.rotary(x, pos, inv)
    for step in (0, 5, 999):
        pos.copy_(i32(np.arange(9) + step))
        graph.replay()
        with torch.cuda.stream(other):
            z = mq.rotary(x, i32(np.arange(9) - step), inv)
        torch.cuda.synchronize()
        within(y, *ref.rotary(f64(x), np.arange(9) + step, freq(32)))
        within(z, *ref.rotary(f64(x), np.arange(9) - step, freq(32)))
