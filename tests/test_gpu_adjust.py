"""Penalties, biases and masks on logits against the 64-bit form.

Tolerance: a 32-bit rounding of each step and the rounding to the type
(oracle.serving.adjust_logits); logits that no step names keep their bits."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, f64, i32, within

pytestmark = pytest.mark.gpu


def logits(T, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (3 * torch.randn(T, V, generator=g)).to(DTYPES[dtype]).cuda()


def case(T, V, n, m, masked, seed):
    r = np.random.default_rng(seed)
    f = lambda *s: r.random(s).astype(np.float32)
    a = {}
    if n:
        h = (r.random((T, n)) ** 3 * V * 1.05).astype(np.int32)  # a few past the row's end
        h[:, ::7] = -1
        a.update(history=h, history_lengths=r.integers(0, n + 1, T).astype(np.int32),
                 prompts=r.integers(0, n + 1, T).astype(np.int32), repetition=1 + f(T) - 0.3, presence=f(T),
                 frequency=f(T) - 0.2)
    if m:
        a.update(bias_ids=r.integers(-2, V + 2, (T, m)).astype(np.int32), bias=f(T, m) * 8 - 4)
    if masked:
        a["mask"] = r.integers(-2 ** 31, 2 ** 31, (T, -(-V // 32))).astype(np.int32)
    return a


def check(x, a, got):
    y, slack, changed = ref.adjust_logits(f64(x), **a)
    within(got, y, slack)
    still = torch.from_numpy(~changed).cuda()
    bits = torch.int32 if x.dtype == torch.float32 else torch.int16
    assert torch.equal(got.view(bits)[still], x.view(bits)[still])


def on_gpu(a):
    return {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in a.items()}


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("T,V,n,m,masked", [
    (1, 1, 1, 1, True), (1, 33, 5, 0, False), (3, 50257, 300, 7, True), (2, 4099, 0, 0, True), (5, 1000, 0, 64, False),
    (1, 151936, 2000, 20, False), (17, 8192, 33, 300, True), (4, 31, 70, 0, True), (300, 257, 3, 2, True),
])
def test_adjust(dtype, T, V, n, m, masked):
    announce("adjust", dtype, T, V, n, m, masked)
    x, a = logits(T, V, dtype, V), case(T, V, n, m, masked, T + V)
    check(x, a, mq.adjust_logits(x, **on_gpu(a)))


@pytest.mark.parametrize("left_out", ["history_lengths", "prompts", "repetition", "presence", "frequency"])
def test_each_part_may_be_left_out(left_out):
    announce("adjust without", left_out)
    x, a = logits(3, 500, "f32", 1), case(3, 500, 40, 0, False, 2)
    del a[left_out]
    check(x, a, mq.adjust_logits(x, **on_gpu(a)))


def test_nothing_to_do_copies():
    announce("adjust nothing")
    x = logits(3, 777, "bf16", 1)
    assert torch.equal(mq.adjust_logits(x), x)
    none = dict(history=torch.zeros(3, 0, dtype=torch.int32, device="cuda"), repetition=torch.ones(3, device="cuda"),
                bias_ids=torch.zeros(3, 0, dtype=torch.int32, device="cuda"), bias=torch.zeros(3, 0, device="cuda"))
    assert torch.equal(mq.adjust_logits(x, **none), x)
    assert mq.adjust_logits(x[:0]).shape == (0, 777) and mq.adjust_logits(x[:, :0]).shape == (3, 0)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_special_values(dtype):
    """NaN and infinities in logits and parameters; a mask that leaves nothing."""
    announce("adjust special", dtype)
    x = logits(4, 70, dtype, 1)
    x[0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0])
    x[1] = -float("inf")
    a = dict(history=np.tile(np.arange(6, dtype=np.int32), (4, 1)), repetition=np.float32([1.5, 1.5, 1, np.inf]),
             presence=np.float32([1, 1, np.inf, 0]), frequency=np.float32([0.5, 0, 0, 0]),
             bias_ids=np.tile(np.int32([0, 69, 5]), (4, 1)), bias=np.float32([[1, 2, -np.inf]] * 4))
    with np.errstate(invalid="ignore"):
        check(x, a, mq.adjust_logits(x, **on_gpu(a)))
        a["mask"] = np.zeros((4, 3), np.int32)
        got = mq.adjust_logits(x, **on_gpu(a))
    assert bool((got == -float("inf")).all())


def test_the_same_token_again_and_again():
    """One token 70000 times (more than 16 bits count), and named by many biases: the last counts."""
    announce("adjust same token")
    x = logits(2, 5000, "f32", 3)
    a = dict(history=np.full((2, 70000), 4097, np.int32), frequency=np.float32([1e-3, 0.25]),
             bias_ids=np.full((2, 1000), 17, np.int32), bias=np.random.default_rng(1).random((2, 1000)).astype(np.float32))
    first = mq.adjust_logits(x, **on_gpu(a))
    check(x, a, first)
    for _ in range(3):
        assert torch.equal(mq.adjust_logits(x, **on_gpu(a)), first)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_views_and_in_place(dtype):
    announce("adjust views", dtype)
    a = case(5, 333, 20, 9, True, 4)
    wide = logits(5, 400, dtype, 5)
    x = wide[:, 3:336]
    g = on_gpu(a)
    # parameters whose rows are wider than what is used
    for name in ("history", "bias_ids", "bias", "mask"):
        t = g[name]
        g[name] = torch.cat([t, t], 1)[:, :t.shape[1]]
    check(x, a, mq.adjust_logits(x, **g))
    turned = x.t().contiguous().t()
    out = torch.empty_like(turned)
    assert out.stride(1) != 1
    assert mq.adjust_logits(turned, **g, out=out) is out
    check(x, a, out)
    before, x0 = wide.clone(), x.clone()
    mq.adjust_logits(x, **g, out=x)
    check(x0, a, x)
    assert torch.equal(wide[:, :3], before[:, :3]) and torch.equal(wide[:, 336:], before[:, 336:])


def test_with_token_logprobs():
    """A grammar's mask before the log probabilities: what it forbids has probability 0; nothing left: -inf."""
    announce("adjust logprobs")
    x = logits(3, 1000, "bf16", 7)
    mask = np.zeros((3, 32), np.int32)
    mask[0, 2], mask[1, :] = 0b1011, -1
    y = mq.adjust_logits(x, mask=torch.from_numpy(mask).cuda())
    _, entropy, top, ids = mq.token_logprobs(y, i32([[64], [5], [1]]), top_k=4)
    assert set(ids[0, :3].tolist()) == {64, 65, 67} and float(top[0, 3]) == -np.inf
    assert abs(float(torch.logsumexp(top[0], 0))) < 1e-5
    assert bool((top[2] == -np.inf).all()) and float(entropy[2]) == 0


def test_graph_of_changing_histories():
    announce("adjust graph")
    x, a = logits(4, 5000, "bf16", 8), case(4, 5000, 50, 5, True, 9)
    g = on_gpu(a)
    mq.adjust_logits(x, **g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mq.adjust_logits(x, **g)
    for seed in (1, 2, 3):
        b = case(4, 5000, 50, 5, True, seed)
        for k, v in on_gpu(b).items():
            g[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        check(x, b, y)
