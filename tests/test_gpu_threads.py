"""Calls of several host threads: on one stream, whose workspaces they share."""
import threading

import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from serving import Cache, i32

pytestmark = pytest.mark.gpu


def turned(t):
    """The same values with the last two axes exchanged in memory."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


def strided_calls():
    """Calls whose operands or scratch take several launches, by name."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    calls = {}
    for i, n in enumerate((40, 900)):
        c = Cache([n, 3], 2, 64, 16, "bf16", n)
        q, args = turned(r(2, 4, 64)), (i32(c.table), i32(c.lengths))
        calls[f"attention {i}"] = lambda q=q, c=c, args=args: mq.paged_attention(q, c.k, c.v, *args)
        x, y, w = turned(r(37, 512)), turned(r(37, 512)), r(512)
        calls[f"norm {i}"] = lambda x=x, y=y, w=w: mq.residual_norm(x, y, pre_weight=w)[1]
        z, tok = turned(r(5, 4000)), i32(np.zeros((5, 1)))
        calls[f"logprobs {i}"] = lambda z=z, tok=tok: mq.token_logprobs(z, tok, top_k=4)[2]
        wq, s, b = mq.quantize(r(256, 1024), 64, 4)
        for rows in (1, 40, 300):
            v = turned(r(rows, 1024)) if rows > 1 else r(1, 1024)
            calls[f"matmul {rows} {i}"] = lambda v=v, p=(wq, s, b): mq.quantized_matmul(v, *p)
    return calls


def test_one_stream_of_two_threads():
    announce("two threads, one stream")
    calls = strided_calls()
    want = {name: f() for name, f in calls.items()}
    torch.cuda.synchronize()
    start, got = threading.Barrier(2), {}

    def work(mine):
        start.wait()
        for rep in range(30):
            for name in mine:
                got[name, rep] = calls[name]()

    names = list(calls)
    threads = [threading.Thread(target=work, args=(names[i::2] + names[1 - i::2][:3],)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert {n for n, _ in got} == set(calls)
    wrong = sorted({n for (n, _), r in got.items() if not torch.equal(r, want[n])})
    assert not wrong, wrong


def test_buffers_freed_beside_calls():
    """`clear_cache` of one thread waits for the launches of the calls under way."""
    announce("clear_cache beside calls")
    calls = strided_calls()
    want = {name: f() for name, f in calls.items()}
    got, done = {}, threading.Event()

    def work():
        for rep in range(200):
            for name, f in calls.items():
                got[name, rep] = f()
        done.set()

    t = threading.Thread(target=work)
    t.start()
    cleared = 0
    while cleared < 10 and not done.is_set():
        mq.clear_cache()
        cleared += 1
    t.join()
    torch.cuda.synchronize()
    assert cleared and mq.get_cache_memory() > 0
    wrong = sorted({n for (n, _), r in got.items() if not torch.equal(r, want[n])})
    assert not wrong, wrong
