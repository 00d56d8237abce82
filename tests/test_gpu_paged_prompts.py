"""The paged decoder of examples/paged_decode.py reading its prompts in chunks:
rotated appends, attention of chunks and of single tokens and logit adjustments as
they are used together, against the same decoder with dense attention over the
whole sequence, float32 norms and float32 products of the dequantized weights.

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
from examples.paged_decode import PagedDecoder  # noqa: E402
from helpers import announce  # noqa: E402
from test_gpu_paged_decode import dense_logits  # noqa: E402

pytestmark = pytest.mark.gpu


def prompts_of(lengths, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 2000, (n,), generator=gen).tolist() for n in lengths]


@pytest.mark.parametrize("chunk", [1, 7, 16, 64])
@pytest.mark.parametrize("lengths", [(5, 33, 17), (1, 48)])
def test_prompts_in_chunks_against_the_dense_decoder(chunk, lengths):
    announce("paged prompts", chunk, lengths)
    prompts = prompts_of(lengths, sum(lengths))
    m = PagedDecoder(seed=len(lengths))
    got = m.read(prompts, chunk).float()
    assert m.lengths[:len(prompts)].tolist() == list(lengths)
    for i, p in enumerate(prompts):
        want = dense_logits(m, p)[-1]
        assert float((got[i] - want).abs().max()) <= 5e-2 * float(want.abs().max())


def test_chunks_follow_single_tokens():
    """A second turn: prompts, steps, then more tokens of some rows beside single ones of others."""
    announce("paged prompts second turn")
    first, more, answer = prompts_of((9, 30, 1), 1), prompts_of((20, 1, 37), 2), prompts_of((4, 4, 4), 3)
    m = PagedDecoder(seed=4)
    m.read(first)
    live = m.rows < 3
    for t in range(4):
        tokens = torch.zeros(len(m.rows), dtype=torch.int64, device="cuda")
        tokens[:3] = torch.tensor([a[t] for a in answer], device="cuda")
        out, granted = m.step(tokens, live)
        assert bool(granted.all())
    for i in range(3):
        want = dense_logits(m, first[i] + answer[i])[-1]
        assert float((out[i].float() - want).abs().max()) <= 5e-2 * float(want.abs().max())
    got = m.read(more, 16).float()
    for i in range(3):
        want = dense_logits(m, first[i] + answer[i] + more[i])[-1]
        assert float((got[i] - want).abs().max()) <= 5e-2 * float(want.abs().max())


def test_penalized_answers():
    announce("paged prompts penalized")
    prompts = prompts_of((5, 33), 7)
    m = PagedDecoder(seed=8)
    answers = m.answer(prompts, ways=3, steps=10, chunk=8, repetition=1.5)
    assert len(answers) == 6 and int((m.refs != 0).sum()) == 0
    for i, tokens, score in answers:
        logits = dense_logits(m, prompts[i] + tokens)[len(prompts[i]) - 1:-1]
        bound = 5e-2 * float(logits.abs().max())
        want = torch.log_softmax(logits, -1)[torch.arange(len(tokens)), torch.tensor(tokens, device="cuda")]
        assert abs(score - float(want.sum())) <= 2 * bound * len(tokens)
        for t in range(1, len(tokens)):
            seen = torch.tensor(sorted(set(prompts[i] + tokens[:t])), device="cuda")
            x = logits[t].clone()
            x[seen] = torch.where(x[seen] > 0, x[seen] / 1.5, x[seen] * 1.5)
            # a penalty stretches an error by 1.5 at most
            assert float(x.max() - x[tokens[t]]) <= 2 * 1.5 * bound
    plain = m.answer(prompts, ways=3, steps=10, chunk=8)
    assert [a[1][0] for a in plain] == [a[1][0] for a in answers]


def test_a_chunk_without_a_page_is_refused():
    announce("paged prompts refused")
    m = PagedDecoder(seed=9, pages=3)
    with pytest.raises(RuntimeError, match="no page left"):
        m.read(prompts_of((20, 40), 10))


def test_the_run_in_a_graph():
    """Reserve, rotated append, chunk attention and adjustments captured once and replayed on."""
    announce("paged prompts graph")
    gen = torch.Generator(device="cuda").manual_seed(11)
    rows, hq, hkv, hd, page, pages, width, new = 3, 8, 2, 64, 16, 40, 12, 5
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(torch.bfloat16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    inv, _ = mq.rotary_frequencies(hd)
    q, k, v = rand(rows * new, hq, hd), rand(rows * new, hkv, hd), rand(rows * new, hkv, hd)
    logits = rand(rows, 1000)
    history, penalty = torch.randint(0, 1000, (rows, 40), dtype=torch.int32, device="cuda", generator=gen), torch.full((rows,), 1.3, device="cuda")
    row = torch.arange(rows, dtype=torch.int32, device="cuda").repeat_interleave(new)
    starts, counts = ints([0, new, 2 * new, 3 * new]), ints([new] * rows)
    place = torch.arange(new, dtype=torch.int32, device="cuda").repeat(rows)

    def fresh():
        pools = [torch.zeros(pages, hkv, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        return pools, torch.full((rows, width), -1, dtype=torch.int32, device="cuda"), ints([0] * rows), ints([0] * pages)

    def turn(pools, table, lengths, refs):
        positions = lengths[row.long()] + place
        mq.cache_reserve(table, lengths, refs, counts, page)
        r = mq.rotary_append(q, k, v, *pools, table, positions, row, inv, lengths=lengths)
        a = mq.paged_attention_chunk(r, *pools, table, lengths, starts)
        return a, mq.adjust_logits(logits, history=history, history_lengths=lengths, repetition=penalty)

    eager = fresh()
    want = [tuple(t.clone() for t in turn(*eager)) for _ in range(6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    state = fresh()
    with torch.cuda.stream(side):
        turn(*state)  # the stream's workspace
        for t in (state[1], *state[0]):
            t.fill_(-1) if t.dtype == torch.int32 else t.zero_()
        state[2].zero_(), state[3].zero_()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = turn(*state)
    for i in range(6):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])
        mq.paged_attention_chunk(q, *state[0], state[1], state[2], starts)  # eager work between replays
