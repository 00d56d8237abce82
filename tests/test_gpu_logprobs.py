"""Token log probabilities, entropy and alternatives against their 64-bit form;
the alternatives' tokens have to be equal."""
import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce
from oracle import serving as ref
from serving import DTYPES, f64, i32, within

pytestmark = pytest.mark.gpu


def check(x, tokens, k, scale=1.0):
    tokens = np.asarray(tokens, np.int32)
    given, ent, top, ids = mq.token_logprobs(x, i32(tokens), top_k=k, scale=scale)
    wg, we, wt, wi, dl, de = ref.token_logprobs(f64(x), tokens, k, float(np.float32(scale)))
    if k:
        np.testing.assert_array_equal(ids.cpu().numpy(), wi)
    else:
        assert top is None and ids is None
    # of the difference z itself, three roundings
    with np.errstate(invalid="ignore"):
        slack = lambda w: np.nan_to_num(dl[:, None] + 4 * ref.U * np.abs(w), posinf=0)
        within(given, wg, slack(wg), "given")
        within(ent, we, de, "entropy")
        if k:
            within(top, wt, slack(wt), "top")


def logits(T, V, dtype, seed, scale=3.0):
    return (scale * torch.randn(T, V, generator=torch.Generator().manual_seed(seed))).to(DTYPES[dtype]).cuda()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 4097, 32000, 50257, 151936])
def test_rows(dtype, V):
    announce("logprobs rows", dtype, V)
    g = np.random.default_rng(V)
    for T, k in ((1, min(V, 20)), (3, min(V, 64))):
        check(logits(T, V, dtype, V + T), g.integers(0, V, (T, 2)), k, 0.7)


@pytest.mark.parametrize("k", [0, 1, 5, 63, 64])
@pytest.mark.parametrize("T", [1, 2, 40, 700])
def test_alternatives(T, k):
    announce("logprobs alternatives", T, k)
    check(logits(T, 3001, "bf16", T + k), np.full((T, 1), 7), k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [64, 3000, 70001])
def test_equal_logits(dtype, V):
    announce("logprobs ties", dtype, V)
    x = torch.zeros(6, V, device="cuda")
    x[1] = -2.5
    x[2, ::2] = -0.0
    x[3] = torch.arange(V, device="cuda") % 3  # a third of the row shares the largest value
    x[4] = torch.finfo(torch.float32).min if dtype == "f32" else float(torch.finfo(torch.bfloat16).min)
    x[5] = torch.arange(V, device="cuda").flip(0) % 7
    check(x.to(DTYPES[dtype]), np.tile([0, V - 1], (6, 1)), min(V, 64), 1.6)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_sorted_rows(dtype):
    announce("logprobs sorted", dtype)
    x = torch.linspace(-20, 20, 5000)
    check(torch.stack([x, x.flip(0)]).to(DTYPES[dtype]).cuda(), [[0], [4999]], 64)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [100, 40000])
def test_masked_and_bad_values(dtype, V):
    announce("logprobs masked", dtype, V)
    inf = float("inf")
    x = logits(8, V, dtype, 3)
    x[0, : V - 3] = -inf  # three tokens left
    x[1] = -inf           # none
    x[2, 5] = inf
    x[3, 7] = float("nan")
    x[4, ::2] = torch.finfo(x.dtype).min
    x[5] = torch.finfo(x.dtype).min
    x[6, 1:] = -inf       # one token left
    x[7, 3] = 80.0        # one token far above the rest
    check(x, np.tile([0, V - 1, V // 2, -1, V, 2 ** 31 - 1, -(2 ** 31)], (8, 1)), 20, 1.3)


@pytest.mark.parametrize("scale", [1e-3, 0.5, 1.0, 30.0])
def test_scales(scale):
    announce("logprobs scale", scale)
    check(logits(3, 20000, "f32", 5), [[1, 2], [3, 4], [5, 6]], 9, scale)


def test_strides_empty_and_no_tokens():
    announce("logprobs strides")
    x = logits(4, 700, "bf16", 6)
    tok = i32([[1, 2]] * 4)
    want = mq.token_logprobs(x, tok, top_k=8)
    wide = torch.zeros(4, 1001, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:703] = x
    for other in (wide[:, 3:703], x.t().contiguous().t()):
        for a, b in zip(mq.token_logprobs(other, tok, top_k=8), want):
            assert torch.equal(a, b)
    given, ent, top, ids = mq.token_logprobs(x[:0], tok[:0], top_k=3)
    assert given.shape == (0, 2) and ent.shape == (0,) and top.shape == ids.shape == (0, 3)
    given, ent, top, ids = mq.token_logprobs(x, torch.empty(4, 0, dtype=torch.int32, device="cuda"), top_k=8)
    assert given.shape == (4, 0) and torch.equal(ids, want[3])


def test_repeatable_graph_and_ctypes(monkeypatch):
    announce("logprobs graph")
    x = logits(2, 60000, "f32", 7)
    tok = i32([[5], [9]])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        mq.token_logprobs(x, tok, top_k=20)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = mq.token_logprobs(x, tok, top_k=20)
    for rep in range(4):
        x.copy_(logits(2, 60000, "f32", 20 + rep))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = mq.token_logprobs(x, tok, top_k=20)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
    from mlxcel_amd import ops

    monkeypatch.setattr(ops, "_native", ops._ctypes_only)
    assert all(torch.equal(a, b) for a, b in zip(mq.token_logprobs(x, tok, top_k=20), want))


@pytest.mark.parametrize("dtype,T", [("bf16", 460), ("f16", 460), ("f32", 230), ("bf16", 700)])
@pytest.mark.parametrize("k", [0, 20])
def test_more_than_the_caches_hold(dtype, T, k):
    """Past 128 MiB the logits are read past the caches; rows of one and of two workgroups."""
    announce("logprobs past the caches", dtype, T, k)
    V = 151937
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, V, generator=g, device="cuda", dtype=DTYPES[dtype]) * 3
    x[3, ::2] = -float("inf")
    x[T - 1, 5:9] = x[T - 1].max()
    assert x.numel() * x.element_size() > 128 << 20
    tok = np.random.default_rng(T).integers(0, V, (T, 2)).astype(np.int32)
    given, ent, top, ids = mq.token_logprobs(x, i32(tok), top_k=k, scale=0.7)
    few = [0, 3, T // 2, T - 1]
    wg, we, wt, wi, dl, de = ref.token_logprobs(f64(x[few]), tok[few], k, float(np.float32(0.7)))
    with np.errstate(invalid="ignore"):
        slack = lambda w: np.nan_to_num(dl[:, None] + 4 * ref.U * np.abs(w), posinf=0)
        within(given[few], wg, slack(wg), "given")
        within(ent[few], we, de, "entropy")
        if k:
            np.testing.assert_array_equal(ids[few].cpu().numpy(), wi)
            within(top[few], wt, slack(wt), "top")
            # every row's alternatives, against a call that leaves the caches as they are
            for r in range(0, T, 100):
                assert torch.equal(mq.token_logprobs(x[r:r + 100], i32(tok[r:r + 100]), top_k=k)[3], ids[r:r + 100])
