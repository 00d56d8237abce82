"""The operators on a cache's pages against their step-by-step form: table,
lengths, references, flags and pools have to be equal, bit for bit."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, i32

pytestmark = pytest.mark.gpu


class Book:
    """A cache with random lengths; the numpy side is the oracle's."""

    def __init__(self, rows, width, pages, page, seed, fill=0.7, pools=2, Hkv=2, D=16, dtype="bf16", most=None,
                 turned=False):
        g = np.random.default_rng(seed)
        self.page, self.pages = page, pages
        order, at = g.permutation(pages), 0
        self.table = np.full((rows, width), -1, np.int32)
        self.lengths = np.zeros(rows, np.int32)
        self.refs = np.zeros(pages, np.int32)
        for r in range(rows):
            n = int(g.integers(0, (most or width * page) + 1))
            h = -(-n // page)
            if at + h > fill * pages:
                continue
            self.table[r, :h] = order[at:at + h]
            self.refs[order[at:at + h]] = 1
            self.lengths[r] = n
            at += h
        shape = (pages, page, Hkv, D) if turned else (pages, Hkv, page, D)
        self.pools = [torch.from_numpy(g.integers(-99, 99, shape).astype(np.float32)).to(DTYPES[dtype])
                      for _ in range(pools)]
        self.dev_pools = [p.cuda() for p in self.pools]
        if turned:
            self.pools = [p.transpose(1, 2) for p in self.pools]
            self.dev_pools = [p.transpose(1, 2) for p in self.dev_pools]
        self.host = [p.float().numpy().copy() for p in self.pools]
        self.t, self.l, self.r = i32(self.table), i32(self.lengths), i32(self.refs)

    def equal(self, what=""):
        for name, dev, host in (("table", self.t, self.table), ("lengths", self.l, self.lengths),
                                ("refs", self.r, self.refs)):
            np.testing.assert_array_equal(dev.cpu().numpy(), host, err_msg=f"{what} {name}")
        for i, (d, h) in enumerate(zip(self.dev_pools, self.host)):
            np.testing.assert_array_equal(d.float().cpu().numpy(), h, err_msg=f"{what} pool {i}")

    def reserve(self, counts):
        counts = np.asarray(counts, np.int32)
        got = mq.cache_reserve(self.t, self.l, self.r, i32(counts), self.page)
        np.testing.assert_array_equal(got.cpu().numpy(), ref.reserve(self.table, self.lengths, self.refs, counts,
                                                                     self.page))

    def fork(self, src, dst):
        got = mq.cache_fork(self.dev_pools, self.t, self.l, self.r, i32(src), i32(dst))
        np.testing.assert_array_equal(got.cpu().numpy(), ref.fork(self.host, self.table, self.lengths, self.refs, src,
                                                                  dst, self.page))

    def free(self, rows):
        mq.cache_free(self.t, self.l, self.r, i32(rows), self.page)
        ref.free(self.table, self.lengths, self.refs, rows, self.page)

    def compact(self):
        got = mq.cache_compact(self.dev_pools, self.t, self.l, self.r)
        assert int(got) == ref.compact(self.host, self.table, self.lengths, self.refs, self.page)


@pytest.mark.parametrize("rows,width,pages,page", [(1, 1, 1, 1), (1, 40, 50, 16), (5, 9, 30, 3), (64, 20, 1000, 16),
                                                   (130, 64, 5000, 8), (1500, 5, 4000, 4), (3, 3000, 9000, 1)])
def test_reserve(rows, width, pages, page):
    announce("reserve", rows, width, pages, page)
    b = Book(rows, width, pages, page, rows + pages)
    g = np.random.default_rng(rows)
    for most in (1, 2 * page, width * page // 2, 1, 0):
        b.reserve(g.integers(0, most + 1, rows))
        b.equal(most)


def test_reserve_with_too_few_pages():
    announce("reserve short")
    for seed in range(6):
        b = Book(1100, 12, 3000, 4, seed, fill=0.97)
        g = np.random.default_rng(seed)
        b.reserve(g.integers(0, 40, 1100))
        b.equal(seed)
        b.reserve(g.integers(0, 9, 1100))
        b.equal(seed)


def test_reserve_refuses_rows():
    announce("reserve refusals")
    b = Book(6, 4, 20, 8, 3, fill=0.5, most=20)
    b.lengths[2] = -3
    b.l.copy_(i32(b.lengths))
    b.reserve([2 ** 31 - 1, 33, 5, -1, 1, 0])
    b.equal()


@pytest.mark.parametrize("dtype,Hkv,D,turned", [("bf16", 2, 16, False), ("f16", 1, 3, False), ("f32", 3, 8, True),
                                                ("bf16", 8, 128, False), ("f32", 1, 5, False)])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [40, 0, 7, 100]])
def test_append(dtype, Hkv, D, turned, counts):
    announce("append", dtype, Hkv, D, counts)
    b = Book(4, 30, 200, 8, 5, fill=0.6, Hkv=Hkv, D=D, dtype=dtype, most=100, turned=turned)
    start = b.lengths.copy()
    b.reserve(counts)
    rows = np.concatenate([np.full(c, r) for r, c in enumerate(counts)])
    pos = np.concatenate([start[r] + np.arange(c) for r, c in enumerate(counts)])
    order = np.random.default_rng(1).permutation(len(rows))
    rows, pos = rows[order], pos[order]
    k, v = (torch.randn(len(rows), Hkv, D).to(DTYPES[dtype]) for _ in range(2))
    for i, (r, p) in enumerate(zip(rows, pos)):
        b.host[0][b.table[r, p // 8], :, p % 8] = k[i].float().numpy()
        b.host[1][b.table[r, p // 8], :, p % 8] = v[i].float().numpy()
    # k as a slice of a wider projection
    wide = torch.randn(len(rows), Hkv, D + 1).to(DTYPES[dtype]).cuda()
    wide[..., :D] = k.cuda()
    mq.cache_append(wide[..., :D], v.cuda(), b.dev_pools[0], b.dev_pools[1], b.t, i32(pos), i32(rows))
    b.equal()


def test_append_leaves_out_what_has_no_place():
    announce("append refusals")
    b = Book(3, 4, 20, 8, 7, fill=0.9, most=20)
    b.table[1, 2:] = [-1, 99]
    b.lengths[:] = [20, 30, 3]
    b.t.copy_(i32(b.table))
    b.l.copy_(i32(b.lengths))
    rows, pos = np.array([0, -1, 3, 1, 1, 0, 2, 0]), np.array([-1, 0, 0, 17, 25, 32, 3, 2 ** 31 - 1])
    k = torch.randn(8, 2, 16).to(torch.bfloat16).cuda()
    b.table[2, 0] = b.table[0, 0]  # a stale entry: its token is past the length
    b.t.copy_(i32(b.table))
    mq.cache_append(k, k, b.dev_pools[0], b.dev_pools[1], b.t, i32(pos), i32(rows), lengths=b.l)
    b.equal()


@pytest.mark.parametrize("dtype,D,turned", [("bf16", 16, False), ("f32", 16, True), ("f16", 3, False)])
@pytest.mark.parametrize("pools", [1, 5, 300])
def test_fork(dtype, D, turned, pools):
    announce("fork", dtype, D, pools)
    b = Book(40, 12, 150, 8, pools + D, fill=0.6, pools=pools, Hkv=1, D=D, dtype=dtype, most=60, turned=turned)
    empty, held = np.flatnonzero(b.lengths == 0), np.flatnonzero(b.lengths)
    src, dst = np.resize(held[:4], len(empty) + 2), np.concatenate([empty, [held[0], -1]])
    b.fork(src, dst)
    b.equal("fork")
    b.free(dst[:len(empty) // 2])
    b.equal("free")
    b.compact()
    b.equal("compact")


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.float64])
@pytest.mark.parametrize("D", [16, 5])
def test_pools_of_any_element(dtype, D):
    """Pages of odd sizes in bytes are moved whole."""
    announce("pools of", dtype, D)
    b = Book(30, 6, 80, 3, D, fill=0.6, pools=0, most=15)
    b.host = [np.random.default_rng(i).integers(0, 200, (80, 1, 3, D)).astype(np.float32) for i in range(3)]
    b.dev_pools = [torch.from_numpy(h).to(dtype).cuda() for h in b.host]
    held, empty = np.flatnonzero(b.lengths), np.flatnonzero(b.lengths == 0)
    b.fork(np.resize(held, len(empty)), empty)
    b.equal("fork")
    b.free(held[::2])
    b.compact()
    b.equal("compact")


def test_many_pages():
    announce("many pages")
    b = Book(300, 90, 60001, 4, 37, fill=0.99, pools=1, Hkv=1, D=2)
    b.reserve(np.random.default_rng(1).integers(0, 300, 300))
    b.equal("reserve")
    b.free(np.arange(0, 300, 2))
    b.compact()
    b.equal("compact")


def test_fork_refusals():
    announce("fork refusals")
    b = Book(12, 6, 24, 4, 11, fill=0.75, most=14)
    held, empty = np.flatnonzero(b.lengths), np.flatnonzero(b.lengths == 0)
    a, e = int(held[0]), [int(x) for x in empty] + [int(held[-1])] * 3
    # one row twice, an empty source, a source that this call makes, rows out of range
    b.fork([a, a, e[0], e[0], 12, a, a], [e[0], e[0], e[1], a, e[1], 99, e[1]])
    b.equal()


def test_fork_with_too_few_pages():
    announce("fork short")
    b = Book(1400, 4, 900, 4, 13, fill=0.9, most=15)
    held, empty = np.flatnonzero(b.lengths), np.flatnonzero(b.lengths == 0)
    b.fork(np.resize(held, len(empty)), empty)
    b.equal()


def test_free_rows_named_twice_and_out_of_range():
    announce("free")
    b = Book(20, 8, 100, 4, 17, fill=0.9)
    b.free([3, 3, 7, -1, 20, 0, 3])
    b.equal()


@pytest.mark.parametrize("rows,width,pages,page,pools", [(1, 1, 1, 1, 1), (20, 10, 120, 4, 3), (200, 12, 2500, 8, 2),
                                                         (4, 3, 5000, 4, 1)])
def test_compact(rows, width, pages, page, pools):
    announce("compact", rows, pages)
    b = Book(rows, width, pages, page, rows + 1, fill=0.95, pools=pools)
    b.compact()
    b.equal("first")
    b.free(np.arange(0, rows, 3))
    b.compact()
    b.equal("second")
    b.compact()  # nothing left to move
    b.equal("third")
    b.free(np.arange(rows))
    b.compact()
    b.equal("empty")


def test_a_life_of_a_cache():
    announce("life")
    g = np.random.default_rng(23)
    b = Book(30, 16, 260, 4, 23, fill=0.3, pools=4, most=20)
    for step in range(12):
        live = b.lengths > 0
        b.reserve(np.where(live, g.integers(0, 7, 30), 0))
        held, empty = np.flatnonzero(b.lengths), np.flatnonzero(b.lengths == 0)
        if len(held) and len(empty):
            n = min(4, len(empty))
            b.fork(g.choice(held, n), empty[:n])
        b.free(g.choice(30, 3))
        if step % 3 == 2:
            b.compact()
        b.equal(step)


def test_graph():
    announce("pages graph")
    b = Book(10, 8, 80, 4, 29, fill=0.4, most=10)
    counts, rows = i32(np.ones(10)), i32([2, 5])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    state = [x.clone() for x in (b.t, b.l, b.r, *b.dev_pools)]
    saved = [x.clone() for x in state]

    def step():
        ok = mq.cache_reserve(state[0], state[1], state[2], counts, 4)
        mq.cache_free(state[0], state[1], state[2], rows, 4)
        return ok, mq.cache_compact(state[3:], *state[:3])

    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    for d, v in zip(state, saved):
        d.copy_(v)
    for rep in range(3):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        b.reserve(np.ones(10))
        b.free([2, 5])
        b.compact()
        b.equal(rep)
        for got, want in zip(state, (b.t, b.l, b.r, *b.dev_pools)):
            assert torch.equal(got, want), rep


def test_the_ctypes_path_gives_the_same(monkeypatch):
    from mlxcel_amd import ops

    monkeypatch.setattr(ops, "_native", ops._ctypes_only)
    b = Book(20, 8, 100, 4, 31, fill=0.6, most=20)
    b.reserve(np.full(20, 3))
    held, empty = np.flatnonzero(b.lengths), np.flatnonzero(b.lengths == 0)
    b.free(held[:3])
    b.fork(held[4:6], held[:2])
    k = torch.randn(1, 2, 16).to(torch.bfloat16)
    r, p = int(held[5]), 0
    mq.cache_append(k.cuda(), k.cuda(), *b.dev_pools, b.t, i32([p]), i32([r]))
    for h in b.host:
        h[b.table[r, 0], :, 0] = k[0].float().numpy()
    b.compact()
    b.equal()


def test_capture_after_a_reserve():
    """On a stream that has run nothing yet."""
    announce("pages capture after a reserve")
    b = Book(10, 8, 80, 4, 29, fill=0.4, most=10)
    held, empty = np.flatnonzero(b.lengths), np.flatnonzero(b.lengths == 0)
    b.free(held[-2:])
    src, dst = held[:2], np.concatenate([held[-2:], empty])[:2]
    counts, s, d = i32(np.ones(10)), i32(src), i32(dst)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        mq.workspace_reserve(1 << 20)
    torch.cuda.synchronize()
    size = mq.get_cache_memory()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        forked = mq.cache_fork(b.dev_pools, b.t, b.l, b.r, s, d)
        granted = mq.cache_reserve(b.t, b.l, b.r, counts, b.page)
        live = mq.cache_compact(b.dev_pools, b.t, b.l, b.r)
    assert mq.get_cache_memory() == size
    for rep in range(3):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = ref.fork(b.host, b.table, b.lengths, b.refs, src, dst, b.page)
        np.testing.assert_array_equal(forked.cpu().numpy(), want)
        assert rep or want.all()
        np.testing.assert_array_equal(granted.cpu().numpy(), ref.reserve(b.table, b.lengths, b.refs, np.ones(10, np.int32),
                                                                         b.page))
        assert int(live) == ref.compact(b.host, b.table, b.lengths, b.refs, b.page)
        b.equal(rep)
