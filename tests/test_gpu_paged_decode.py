"""The paged decoder of examples/paged_decode.py against the same decoder with
dense attention over the whole sequence, float32 norms and float32 products of
the dequantized weights: the log probabilities of its answers, which pass
through forks, frees and a compaction.

The bound 5e-2 is the decoder's of test_gpu_e2e.py (whole networks in bfloat16
on both sides), here relative to the largest logit.
"""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import mlxcel_amd as mq  # noqa: E402
from examples.paged_decode import BITS, GS, PagedDecoder  # noqa: E402
from helpers import announce  # noqa: E402

pytestmark = pytest.mark.gpu


def dense_logits(m, tokens):
    """Logits after every token of one sequence."""
    bf = lambda t: t.to(torch.bfloat16)

    def mm(x, w):
        return bf(x.float() @ mq.dequantize(*w, GS, BITS).float().t())

    def rms(t, w):
        t = t.float()
        return t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w.float()

    n, G = len(tokens), m.nq // m.nkv
    pos = torch.arange(n, device="cuda")
    h = m.embed[torch.tensor(tokens, device="cuda")]
    mask = torch.full((n, n), float("-inf"), device="cuda").triu(1)
    for L in m.layers:
        x = bf(rms(h, L["pre"]))
        q, k, v = (mm(x, w).view(n, -1, m.hd) for w in L["qkv"])
        q, k = m.rope(q, pos), m.rope(k, pos)
        q, k, v = (t.float().transpose(0, 1).contiguous() for t in (q, k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)))
        p = torch.softmax(torch.matmul(q, k.transpose(1, 2).contiguous()) * m.hd ** -0.5 + mask, -1)
        a = bf(torch.matmul(p, v).transpose(0, 1).reshape(n, -1))
        h = bf(h.float() + rms(mm(a, L["o"]), L["post"]))
        x = bf(rms(h, L["mid"]))
        g, u = (mm(x, w).float() for w in L["gu"])
        h = bf(h.float() + mm(bf(torch.nn.functional.silu(g) * u), L["d"]).float())
    return mm(bf(rms(h, m.last)), m.lm).float()


@pytest.mark.parametrize("lengths", [(5, 33, 17), (16,), (1, 48)])
def test_answers_against_the_dense_decoder(lengths):
    announce("paged decode", lengths)
    gen = torch.Generator().manual_seed(sum(lengths))
    prompts = [torch.randint(0, 2000, (n,), generator=gen).tolist() for n in lengths]
    m = PagedDecoder(seed=len(lengths))
    answers = m.answer(prompts, ways=3, steps=10)
    assert len(answers) == 3 * len(prompts)
    assert int((m.refs != 0).sum()) == 0 and int(m.lengths.abs().sum()) == 0
    for i, tokens, score in answers:
        logits = dense_logits(m, prompts[i] + tokens)[len(prompts[i]) - 1:-1]
        lp = torch.log_softmax(logits, -1)
        want = lp[torch.arange(len(tokens)), torch.tensor(tokens, device="cuda")]
        bound = 5e-2 * float(logits.abs().max())
        # each chosen token is the greatest within the bound (the first: among the greatest three)
        for t in range(1, len(tokens)):
            assert float(lp[t].max() - want[t]) <= 2 * bound
        assert abs(score - float(want.sum())) <= 2 * bound * len(tokens)


def test_steps_are_the_same_after_compaction():
    announce("paged decode compaction")
    m = PagedDecoder(seed=5)
    gen = torch.Generator().manual_seed(6)
    live = torch.zeros(16, dtype=torch.bool, device="cuda")
    live[:6] = True
    for _ in range(40):
        m.step(torch.randint(0, 2000, (16,), generator=gen).cuda(), live)
    mq.cache_free(m.table, m.lengths, m.refs, m.rows[1:4], m.page)
    live[1:4] = False
    state = [t.clone() for t in (m.table, m.lengths, m.refs, *m.pools)]
    tokens = torch.randint(0, 2000, (16,), generator=gen).cuda()
    want, _ = m.step(tokens, live)
    for t, s in zip((m.table, m.lengths, m.refs, *m.pools), state):
        t.copy_(s)
    before = m.table.clone()
    live_pages = int(mq.cache_compact(m.pools, m.table, m.lengths, m.refs))
    assert live_pages == 9 and not torch.equal(before, m.table)
    got, _ = m.step(tokens, live)
    assert torch.equal(got[live], want[live])
