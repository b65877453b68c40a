"""The largest launches of the sequence-layer operators (tests/test_seq_limits.py has what is refused): their last rows come out as when
they are given alone."""
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

MOST = (2 ** 32 - 1) // 256   # workgroups of 256 threads
BF16 = torch.bfloat16


def _rows(n, *shape):
    """n rows, random ones among zeros at both ends."""
    x = torch.zeros(n, *shape, device='cuda')
    x[:50], x[-50:] = (torch.randn(50, *shape, generator=torch.Generator().manual_seed(s)).cuda() for s in (131, 132))
    return x


def test_the_most_sequences():
    from blocks.delta_rule import gated_delta_rule
    q, k, v = (_rows(MOST, 2, 1, 1).to(BF16) for _ in range(3))
    g, beta = -_rows(MOST, 2, 1).abs(), _rows(MOST, 2, 1).sigmoid()
    o, final = gated_delta_rule(q, k, v, g, beta)
    for at in (slice(0, 50), slice(-50, None)):
        lo, lf = gated_delta_rule(*(x[at] for x in (q, k, v, g, beta)))
        assert torch.equal(o[at], lo) and torch.equal(final[at], lf) and (lo != 0).any()


def test_the_most_single_tokens():
    from blocks.delta_rule import gated_delta_step
    q, k, v = (_rows(MOST, 1, 1).to(BF16) for _ in range(3))
    g, beta, state = -_rows(MOST, 1).abs(), _rows(MOST, 1).sigmoid(), _rows(MOST, 1, 1, 1)
    was = state.clone()
    o = gated_delta_step(q, k, v, g, beta, state)
    for at in (slice(0, 50), slice(-50, None)):
        own = was[at].clone()
        assert torch.equal(gated_delta_step(*(x[at] for x in (q, k, v, g, beta)), own), o[at]) and torch.equal(own, state[at])


def test_the_most_rows_of_a_unit():
    from blocks.gated_unit import gated_unit
    M = 2 ** 30 - 256
    x = torch.zeros(M, 8, device='cuda', dtype=BF16)
    x[-300:] = torch.randn(300, 8, generator=torch.Generator().manual_seed(133)).cuda()
    wg, wu = (torch.randn(8, 8, generator=torch.Generator().manual_seed(s)).cuda().to(BF16) for s in (134, 135))
    y = gated_unit(x, wg, wu)
    assert torch.equal(y[-300:], gated_unit(x[-300:], wg, wu)) and (y[-300:] != 0).any() and not y[:1000].any()
