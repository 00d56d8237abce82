"""The paged decoder of examples/paged_decode.py looks at a step's logits as often as
its answers need: once without penalties, twice with them (for the choice, and
for the log probability that the logits give what was chosen)."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import mlxcel_amd as mq  # noqa: E402
from examples.paged_decode import PagedDecoder  # noqa: E402
from helpers import announce  # noqa: E402
from test_gpu_paged_prompts import prompts_of  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("repetition,passes", [(1.0, 1), (1.3, 2)])
def test_passes_over_the_logits(monkeypatch, repetition, passes):
    announce("paged passes", repetition)
    calls, steps, prompts = [], 9, prompts_of((5, 20), 3)
    plain = mq.token_logprobs
    monkeypatch.setattr(mq, "token_logprobs", lambda *a, **kw: calls.append(a[0].shape) or plain(*a, **kw))
    m = PagedDecoder(seed=5)
    answers = m.answer(prompts, ways=2, steps=steps, repetition=repetition)
    assert len(calls) == 1 + passes * (steps - 1)
    assert len(answers) == 4 and all(len(tokens) == steps for _, tokens, _ in answers)
