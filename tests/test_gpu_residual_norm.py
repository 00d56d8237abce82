"""The residual update and its norms against their 64-bit form."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, f64, within

pytestmark = pytest.mark.gpu


def rnd(shape, dtype, seed, scale=1.0):
    return (scale * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def check(x, y, post=None, gate=None, scale=1.0, pre=None, eps=1e-6, offset=0.0):
    h, n = mq.residual_norm(x, y, post_weight=post, gate=gate, scale=scale, pre_weight=pre, eps=eps,
                            weight_offset=offset)
    o = [None if t is None else f64(t) for t in (post, gate, pre)]
    f = lambda v: float(np.float32(v))
    wh, dh, wn, dn = ref.residual_norm(f64(x), f64(y), o[0], o[1], f(scale), o[2], f(eps), f(offset))
    within(h, wh, dh, "h")
    if pre is None:
        assert n is None
    else:
        within(n, wn, dn, "n")
    return h, n


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H", [1, 7, 8, 63, 64, 100, 255, 1000, 1152, 2049, 4096, 5121, 8192, 12001, 32768])
def test_widths(dtype, H):
    announce("norm widths", dtype, H)
    dt = DTYPES[dtype]
    for T in (1, 5):
        x, y = rnd((T, H), dt, H), rnd((T, H), dt, H + 1, 3.0)
        post, pre = rnd(H, dt, H + 2), rnd(H, dt, H + 3)
        check(x, y, post, rnd((T, H), dt, H + 4), 0.22, pre, offset=1.0)
        check(x, y, pre=pre)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "token", "row", "one", "batch"])
@pytest.mark.parametrize("pre", [False, True])
def test_forms(dtype, post, gate, pre):
    announce("norm forms", dtype, post, gate, pre)
    dt, H = DTYPES[dtype], 136
    x, y = rnd((3, 5, H), dt, 1), rnd((3, 5, H), dt, 2)
    shape = {"channel": (H,), "token": (3, 5, H), "row": (3, 5, 1), "one": (1,), "batch": (3, 1, H)}.get(gate)
    check(x, y, rnd(H, dt, 3) if post else None, rnd(shape, dt, 4) if gate else None, 1.4, rnd(H, dt, 5) if pre else None,
          offset=0.5)


def test_float32_weights_of_16_bit_rows():
    announce("norm f32 weights")
    for dt in (torch.bfloat16, torch.float16):
        x, y = rnd((4, 72), dt, 1), rnd((4, 72), dt, 2)
        check(x, y, rnd(72, torch.float32, 3), None, 1.0, rnd(72, torch.float32, 4))


@pytest.mark.parametrize("rows", [1, 2, 255, 4097])
@pytest.mark.parametrize("H", [64, 200, 2880])
def test_rows(rows, H):
    announce("norm rows", rows, H)
    x, y = rnd((rows, H), torch.bfloat16, 1), rnd((rows, H), torch.bfloat16, 2)
    check(x, y, None, rnd((rows, 1), torch.bfloat16, 3), 0.5, rnd(H, torch.bfloat16, 4))


def test_strides():
    announce("norm strides")
    wide = rnd((6, 300), torch.bfloat16, 1)
    x, y = wide[::2, 3:131], wide[1::2, 101:229]
    w = rnd(128, torch.bfloat16, 2)
    want = mq.residual_norm(x.contiguous(), y.contiguous(), pre_weight=w)
    for a, b in ((x, y), (x.t().contiguous().t(), y), (x, y.t().contiguous().t())):
        got = mq.residual_norm(a, b, pre_weight=w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    row = rnd((1, 128), torch.bfloat16, 3)  # one row, broadcast to all
    check(x, row.expand(3, 128), pre=w, gate=rnd((3, 128, 2), torch.bfloat16, 4)[..., 0])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_of_zeros_large_and_small_values(dtype):
    announce("norm extremes", dtype)
    dt = DTYPES[dtype]
    x, y = torch.zeros(4, 96, dtype=dt, device="cuda"), torch.zeros(4, 96, dtype=dt, device="cuda")
    x[1], y[1] = rnd(96, dt, 1, 100.0), rnd(96, dt, 2, 100.0)
    x[2], y[2] = rnd(96, dt, 3, 1e-3), rnd(96, dt, 4, 1e-3)
    x[3, 5] = 200.0
    check(x, y, rnd(96, dt, 5), None, 1.0, rnd(96, dt, 6))
    y[0, 3] = float("inf")
    y[2, 1] = float("nan")
    h, n = mq.residual_norm(x, y, pre_weight=rnd(96, dt, 7))
    assert torch.isnan(n[2]).all() and torch.isinf(h[0, 3]) and not torch.isnan(n[[1, 3]]).any()
    assert torch.equal(h[[1, 3]], (x.float() + y.float()).to(dt)[[1, 3]])


def test_empty_graph_stream_and_ctypes(monkeypatch):
    announce("norm graph")
    w = rnd(64, torch.bfloat16, 1)
    e = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    h, n = mq.residual_norm(e, e, pre_weight=w)
    assert h.shape == n.shape == (0, 64)
    x, y = rnd((9, 64), torch.bfloat16, 2), rnd((9, 64), torch.bfloat16, 3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = mq.residual_norm(x, y, pre_weight=w, scale=0.5)
    for rep in range(3):
        x.copy_(rnd((9, 64), torch.bfloat16, 10 + rep))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = mq.residual_norm(x, y, pre_weight=w, scale=0.5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    from mlxcel_amd import ops

    monkeypatch.setattr(ops, "_native", ops._ctypes_only)
    again = mq.residual_norm(x, y, pre_weight=w, scale=0.5)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_copies_take_their_own_size():
    """Only what is copied counts: a gate of every other element beside rows of 32 MiB, then the rows too."""
    announce("norm staging size")
    T, H, mib = 2048, 4096, 1 << 20
    x, gate = torch.randn(T, H, device="cuda"), torch.randn(2 * H, device="cuda")[::2]
    want = mq.residual_norm(x, x, gate=gate.contiguous())[0]
    turned = x.t().contiguous().t()
    torch.cuda.synchronize()
    mq.clear_cache()
    assert torch.equal(mq.residual_norm(x, x, gate=gate)[0], want)
    assert mq.get_cache_memory() == mib
    mq.clear_cache()
    assert torch.equal(mq.residual_norm(turned, x, gate=gate)[0], want)
    assert mq.get_cache_memory() == 64 * mib
    mq.clear_cache()
    assert torch.equal(mq.residual_norm(x, turned)[0], mq.residual_norm(x, x)[0])
    assert mq.get_cache_memory() == 32 * mib
