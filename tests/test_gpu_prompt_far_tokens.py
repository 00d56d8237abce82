"""Rotation of as many tokens as a call takes: 2^31 - 1.

The kernel's workgroups go from token to token in steps of 2^20, so a token's
number counted in 31 bits would pass the end of the range in the last step."""
import pytest
import torch

import mlxcel_amd as mq
from helpers import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [2 ** 31 - 1, 2 ** 31 - 2 ** 20 + 1])
def test_rotary_of_the_most_tokens(T):
    """One token's elements for all of them (a stride of 0), positions that come again every 1000 tokens."""
    announce("rotary tokens", T)
    period = 1000
    inv = torch.tensor([0.01], device="cuda")
    x = torch.tensor([[[1.5, -0.75]]], dtype=torch.bfloat16, device="cuda").expand(T, 1, 2)
    pos = torch.empty(T, dtype=torch.int32, device="cuda")
    torch.arange(period, dtype=torch.int32, device="cuda", out=pos[:period])
    whole = T // period * period
    pos[:whole].view(-1, period)[1:] = pos[:period]
    pos[whole:] = pos[:T - whole]
    out = torch.full((T + 2, 1, 2), 7.0, dtype=torch.bfloat16, device="cuda")
    mq.rotary(x, pos, inv, out=out[1:T + 1])
    assert bool((out[0] == 7).all()) and bool((out[T + 1] == 7).all())
    want = mq.rotary(x[:period], pos[:period], inv)
    got = out[1:T + 1]
    block = 10 ** 8
    for at in range(0, whole, block):
        part = got[at:min(at + block, whole)].view(-1, period, 1, 2)
        assert bool((part == want).all()), at
    assert torch.equal(got[whole:], want[:T - whole])
