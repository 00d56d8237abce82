"""CPU checks of the serving operators' arguments (only calls that fail before
any device work), of their Python wrappers' refusals and of their 64-bit forms."""
import ctypes

import numpy as np
import pytest
import torch

import mlxcel_amd as mq
from mlxcel_amd import _lib
from oracle import serving as ref
from test_abi import arr

BF, F16, F32, F64, I32, I64 = _lib.BFLOAT16, _lib.FLOAT16, _lib.FLOAT32, _lib.FLOAT64, _lib.INT32, _lib.INT64
EINVAL, EUNSUPPORTED = _lib.EINVAL, _lib.EUNSUPPORTED


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def have(shape, dtype, strides=None, data=4096):
    """An array whose data pointer is never followed: the call has to fail."""
    a = arr(shape, dtype, strides)
    a.data = data
    return a


def call(lib, name, *args):
    vals = [ctypes.byref(a) if isinstance(a, _lib.MlxqArray) else a for a in args]
    return getattr(lib, name)(*vals, None), _lib.last_error()


def refused(lib, name, code, text, *args):
    st, msg = call(lib, name, *args)
    assert st == code and text in msg, (st, msg)


ATTN = dict(q=((2, 8, 64), BF), k=((9, 2, 16, 64), BF), v=((9, 2, 16, 64), BF), table=((2, 5), I32), lengths=((2,), I32),
            sinks=None, scale=0.125, softcap=0.0, window=0, out=((2, 8, 64), BF))


@pytest.mark.parametrize("change,code,text", [
    (dict(q=((2, 8), BF)), EINVAL, "q must have 3 dimensions"),
    (dict(q=((2, 8, 64), F64)), EINVAL, "bfloat16, float16 or float32 but is float64"),
    (dict(k=((9, 2, 16, 64), F16)), EINVAL, "k_pool must be bfloat16"),
    (dict(v=((9, 2, 8, 64), BF)), EINVAL, "v_pool must have shape"),
    (dict(q=((2, 7, 64), BF)), EINVAL, "query heads (7)"),
    (dict(q=((2, 8, 72), BF)), EINVAL, "one head width"),
    (dict(table=((3, 5), I32)), EINVAL, "one row a sequence"),
    (dict(table=((2, 5), I64)), EINVAL, "table must be int32"),
    (dict(table=((2, 5), I32, (1, 2))), EUNSUPPORTED, "rows must be contiguous"),
    (dict(table=((2, 1 << 27), I32)), EUNSUPPORTED, "too wide"),
    (dict(lengths=((2,), I32, (2,))), EUNSUPPORTED, "lengths must be contiguous"),
    (dict(sinks=((7,), F32)), EINVAL, "sinks must have shape"),
    (dict(sinks=((8,), BF)), EINVAL, "sinks must be float32"),
    (dict(scale=float("nan")), EINVAL, "scale"),
    (dict(softcap=-1.0), EINVAL, "softcap"),
    (dict(softcap=float("inf")), EINVAL, "softcap"),
    (dict(window=-1), EINVAL, "window"),
    (dict(out=((2, 8, 64), F32)), EINVAL, "out must have shape"),
    (dict(k=((9, 2, 16, 64), BF, (2048, 1024, 1, 16))), EUNSUPPORTED, "last axis must be contiguous"),
    (dict(k=((0, 2, 16, 64), BF), v=((0, 2, 16, 64), BF)), EINVAL, "no pages"),
    (dict(q=((2, 8, 60), BF), k=((9, 2, 16, 60), BF), v=((9, 2, 16, 60), BF), out=((2, 8, 60), BF)), EUNSUPPORTED,
     "multiple of 8"),
    (dict(q=((2, 8, 264), BF), k=((9, 2, 16, 264), BF), v=((9, 2, 16, 264), BF), out=((2, 8, 264), BF)), EUNSUPPORTED,
     "up to 256"),
])
def test_paged_attention(lib, change, code, text):
    a = {**ATTN, **change}
    refused(lib, "mlxq_paged_attention", code, text, *[have(*v) if isinstance(v, tuple) else v for v in a.values()])


def test_data_pointers(lib):
    a = {k: have(*v) if isinstance(v, tuple) else v for k, v in ATTN.items()}
    refused(lib, "mlxq_paged_attention", EINVAL, "k_pool has no data", *{**a, "k": arr((9, 2, 16, 64), BF)}.values())
    refused(lib, "mlxq_paged_attention", EINVAL, "not aligned", *{**a, "q": have((2, 8, 64), BF, None, 4097)}.values())
    refused(lib, "mlxq_paged_attention", EINVAL, "must not be NULL", *{**a, "table": None}.values())


BOOK = [have((4, 6), I32), have((4,), I32), have((20,), I32)]


@pytest.mark.parametrize("args,code,text", [
    ([*BOOK, have((3,), I32), 16, have((4,), I32)], EINVAL, "counts must have shape"),
    ([*BOOK, have((4,), I32), 0, have((4,), I32)], EINVAL, "at least one token"),
    ([*BOOK, have((4,), I32), 1 << 28, have((4,), I32)], EUNSUPPORTED, "too wide"),
    ([*BOOK, have((4,), I32), 16, have((4,), F32)], EINVAL, "granted must be int32"),
    ([BOOK[0], BOOK[1], have(((1 << 30) + 1,), I32), have((4,), I32), 16, have((4,), I32)], EUNSUPPORTED, "too many pages"),
    ([BOOK[0], have((5,), I32), BOOK[2], have((4,), I32), 16, have((4,), I32)], EINVAL, "as many rows"),
])
def test_cache_reserve(lib, args, code, text):
    refused(lib, "mlxq_cache_reserve", code, text, *args)


def pools(*arrays):
    P = ctypes.POINTER(_lib.MlxqArray)
    return (P * len(arrays))(*[ctypes.pointer(a) for a in arrays])


POOL = have((20, 2, 16, 8), BF)


@pytest.mark.parametrize("n,list_,code,text", [
    (0, pools(POOL), EINVAL, "at least one pool"),
    (2, pools(POOL, have((20, 2, 16, 8), F16)), EINVAL, "one shape and type"),
    (1, pools(have((21, 2, 16, 8), BF)), EINVAL, "one entry a page"),
    (1, pools(have((20, 2, 16), BF)), EINVAL, "4 dimensions"),
    (1, pools(have((20, 2, 16, 8), BF, (512, 256, 16, 2))), EUNSUPPORTED, "dense block"),
    (2, pools(POOL, have((20, 2, 16, 8), BF, (512, 128, 8, 1))), EUNSUPPORTED, "same strides"),
])
def test_pools(lib, n, list_, code, text):
    refused(lib, "mlxq_cache_fork", code, text, n, list_, *BOOK, have((2,), I32), have((2,), I32), have((2,), I32))
    refused(lib, "mlxq_cache_compact", code, text, n, list_, *BOOK, have((1,), I32))


def test_fork_free_and_compact(lib):
    two = have((2,), I32)
    refused(lib, "mlxq_cache_fork", EINVAL, "dst must have shape", 1, pools(POOL), *BOOK, two, have((3,), I32), two)
    refused(lib, "mlxq_cache_compact", EINVAL, "live must have shape", 1, pools(POOL), *BOOK, two)
    refused(lib, "mlxq_cache_free", EINVAL, "rows must be int32", *BOOK, have((2,), I64), 16)
    refused(lib, "mlxq_cache_free", EINVAL, "1 dimensions", *BOOK, have((2, 1), I32), 16)


def test_forks_and_compactions_of_more_than_a_launch(lib):
    """Refused before the plan, which would have changed the book."""
    many, long = have((1 << 21,), I32), [have((1 << 24, 6), I32), have((1 << 24,), I32), BOOK[2]]
    refused(lib, "mlxq_cache_fork", EUNSUPPORTED, "too many pairs", 1, pools(POOL), *BOOK, many, many, many)
    refused(lib, "mlxq_cache_fork", EUNSUPPORTED, "too many pairs", 300, pools(*[POOL] * 300), *BOOK,
            *[have((1 << 16,), I32)] * 3)
    refused(lib, "mlxq_cache_compact", EUNSUPPORTED, "too long", 1, pools(POOL), *long, have((1,), I32))


APPEND = [have((3, 2, 8), BF), have((3, 2, 8), BF), POOL, POOL, have((4, 6), I32), have((3,), I32), have((3,), I32), None]


@pytest.mark.parametrize("at,a,code,text", [
    (0, have((3, 2, 8), I32), EINVAL, "must be bfloat16"),
    (1, have((3, 2, 9), BF), EINVAL, "v must have shape"),
    (2, have((20, 3, 16, 8), BF), EINVAL, "v_pool must have shape"),
    (5, have((4,), I32), EINVAL, "positions must have shape"),
    (6, have((3,), I64), EINVAL, "rows must be int32"),
    (7, have((3,), I32), EINVAL, "lengths must have shape"),
    (0, have((3, 2, 8), BF, (16, 1, 2)), EUNSUPPORTED, "must be contiguous"),
])
def test_cache_append(lib, at, a, code, text):
    args = list(APPEND)
    args[at] = a
    refused(lib, "mlxq_cache_append", code, text, *args)


NORM = dict(x=((3, 8), BF), y=((3, 8), BF), post=None, gate=None, scale=1.0, pre=((8,), BF), eps=1e-6, off=0.0,
            h=((3, 8), BF), n=((3, 8), BF))


@pytest.mark.parametrize("change,code,text", [
    (dict(x=((), BF)), EINVAL, "at least one dimension"),
    (dict(y=((3, 9), BF)), EINVAL, "y must have shape"),
    (dict(y=((3, 8), F32)), EINVAL, "y must be bfloat16"),
    (dict(post=((9,), BF)), EINVAL, "post_weight must have shape"),
    (dict(pre=((8,), F16)), EINVAL, "or float32"),
    (dict(pre=None), EINVAL, "n is given"),
    (dict(n=None), EINVAL, "n is given"),
    (dict(gate=((), BF)), EINVAL, "at least one dimension"),
    (dict(gate=((2, 8), BF)), EINVAL, "does not broadcast"),
    (dict(gate=((3, 2), BF)), EINVAL, "does not broadcast"),
    (dict(gate=((1, 3, 8), BF)), EINVAL, "more dimensions"),
    (dict(x=((2, 3, 8), BF), y=((2, 3, 8), BF), gate=((1, 3, 8), BF), h=((2, 3, 8), BF), n=((2, 3, 8), BF)),
     EUNSUPPORTED, "broadcast over an axis"),
    (dict(scale=float("inf")), EINVAL, "scale"),
    (dict(eps=-1.0), EINVAL, "eps"),
    (dict(off=float("nan")), EINVAL, "weight_offset"),
    (dict(h=((3, 8), F32)), EINVAL, "out must have shape"),
    (dict(x=((1, 40000), BF), y=((1, 40000), BF), pre=((40000,), BF), h=((1, 40000), BF), n=((1, 40000), BF)),
     EUNSUPPORTED, "at most 32768"),
])
def test_residual_norm(lib, change, code, text):
    a = {**NORM, **change}
    refused(lib, "mlxq_residual_norm", code, text, *[have(*v) if isinstance(v, tuple) else v for v in a.values()])


LOGP = dict(x=((3, 100), BF), tok=((3, 2), I32), k=4, scale=1.0, lp=((3, 2), F32), ent=((3,), F32), top=((3, 4), F32),
            ids=((3, 4), I32))


@pytest.mark.parametrize("change,code,text", [
    (dict(x=((3, 100), I32)), EINVAL, "must be bfloat16"),
    (dict(x=((100,), BF)), EINVAL, "2 dimensions"),
    (dict(tok=((2, 2), I32)), EINVAL, "one row"),
    (dict(tok=((3, 2), I64)), EINVAL, "tokens must be int32"),
    (dict(k=-1), EINVAL, "top_k"),
    (dict(k=101), EINVAL, "top_k"),
    (dict(k=65, top=((3, 65), F32), ids=((3, 65), I32)), EUNSUPPORTED, "at most 64"),
    (dict(scale=0.0), EINVAL, "scale"),
    (dict(scale=-1.0), EINVAL, "scale"),
    (dict(scale=float("nan")), EINVAL, "scale"),
    (dict(lp=((3, 2), BF)), EINVAL, "out must have shape"),
    (dict(ids=((3, 4), I64)), EINVAL, "out must have shape"),
    (dict(top=None), EINVAL, "must not be NULL"),
])
def test_token_logprobs(lib, change, code, text):
    a = {**LOGP, **change}
    refused(lib, "mlxq_token_logprobs", code, text, *[have(*v) if isinstance(v, tuple) else v for v in a.values()])


def test_wrappers_refuse_tensors_off_the_device():
    x, i = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        mq.paged_attention(torch.zeros(2, 2, 8), torch.zeros(1, 1, 4, 8), torch.zeros(1, 1, 4, 8), i[:, None], i)
    with pytest.raises(ValueError, match="HIP device"):
        mq.residual_norm(x, x)
    with pytest.raises(ValueError, match="HIP device"):
        mq.token_logprobs(x, i[:, None], top_k=1)
    for f in (lambda: mq.cache_reserve(i[:, None], i, i, i, 4), lambda: mq.cache_free(i[:, None], i, i, i, 4),
              lambda: mq.cache_fork([torch.zeros(2, 1, 4, 8)], i[:, None], i, i, i, i),
              lambda: mq.cache_compact([torch.zeros(2, 1, 4, 8)], i[:, None], i, i),
              lambda: mq.cache_append(x[:, None], x[:, None], x, x, i[:, None], i, i)):
        with pytest.raises(ValueError, match="HIP device"):
            f()


# ---- the 64-bit forms ---------------------------------------------------------------


def test_attention_form():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((1, 4, 8), (5, 2, 4, 8), (5, 2, 4, 8)))
    table, n = np.array([[3, 0, 4]]), 10
    got, slack = ref.attention(q.numpy(), k.numpy(), v.numpy(), table, [n], 0.5)
    flat = lambda t: t[table[0]].transpose(0, 1).reshape(2, 12, 8)[:, :n].repeat_interleave(2, 0)
    want = torch.nn.functional.scaled_dot_product_attention(q[0][:, None], flat(k), flat(v), scale=0.5)[:, 0]
    np.testing.assert_allclose(got[0], want.numpy(), rtol=1e-12)
    assert 0 < slack.max() < 1e-4
    last, _ = ref.attention(q.numpy(), k.numpy(), v.numpy(), table, [n], 0.5, window=1)
    np.testing.assert_allclose(last[0], flat(v)[:, -1].numpy(), rtol=1e-12)
    none, _ = ref.attention(q.numpy(), k.numpy(), v.numpy(), table, [0], 0.5, sinks=np.zeros(4))
    assert not none.any()


def test_logprobs_form():
    x = np.array([[0.0, 2.0, -np.inf, 2.0, 1.0], [-np.inf] * 5, [np.nan, 1, 0, np.nan, 3]])
    given, ent, top, ids, dl, de = ref.token_logprobs(x, np.array([[1, 2, 9]] * 3), 4, 1.0)
    want = torch.log_softmax(torch.from_numpy(x[0]), 0).numpy()
    np.testing.assert_allclose(top[0], want[[1, 3, 4, 0]], rtol=1e-12)
    assert ids.tolist() == [[1, 3, 4, 0], [0, 1, 2, 3], [0, 3, 4, 1]]
    assert given[0, 1] == -np.inf and np.isnan(given[:, 2]).all() and ent[1] == 0 and np.isnan(ent[2])
    p = np.exp(want)
    np.testing.assert_allclose(ent[0], -(p[p > 0] * want[p > 0]).sum(), rtol=1e-12)


def test_norm_form():
    g = np.random.default_rng(2)
    x, y, w = g.normal(size=(2, 6)), g.normal(size=(2, 6)), g.normal(size=6)
    h, dh, n, dn = ref.residual_norm(x, y, w, None, 0.5, w, 1e-6, 1.0)
    rms = lambda t: torch.nn.functional.rms_norm(torch.from_numpy(t), (6,), torch.from_numpy(w + 1), 1e-6).numpy()
    np.testing.assert_allclose(h, x + 0.5 * rms(y), rtol=1e-12)
    np.testing.assert_allclose(n, rms(h), rtol=1e-12)
    assert (dn > 0).all() and (dh > 0).all()


def test_page_forms_keep_their_invariants():
    g = np.random.default_rng(3)
    table, lengths, refs = np.full((8, 5), -1, np.int32), np.zeros(8, np.int32), np.zeros(25, np.int32)
    pool = g.normal(size=(25, 1, 4, 1))
    for _ in range(40):
        ref.reserve(table, lengths, refs, np.where(g.random(8) < 0.5, g.integers(0, 8, 8), 0), 4)
        held, empty = np.flatnonzero(lengths), np.flatnonzero(lengths == 0)
        if len(held) and len(empty):
            ref.fork([pool], table, lengths, refs, held[:1], empty[:1], 4)
        rows = g.choice(8, 2)
        before = {r: [pool[p] for p in table[r, :-(-lengths[r] // 4)]] for r in range(8)}
        kept = lengths.copy()
        ref.free(table, lengths, refs, rows, 4)
        n = ref.compact([pool], table, lengths, refs, 4)
        assert (refs[:n] > 0).all() and not refs[n:].any()
        count = np.zeros(25, int)
        for r in range(8):
            assert lengths[r] == (0 if r in rows else kept[r])
            for j in range(-(-lengths[r] // 4)):
                count[table[r, j]] += 1
                assert np.array_equal(pool[table[r, j]], before[r][j])
        assert np.array_equal(count, refs)
