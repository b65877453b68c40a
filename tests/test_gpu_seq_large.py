"""Tensors of more than 2^31 elements: the last rows and heads come out as when they are given alone."""
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_a_pool_of_many_states():
    from blocks import delta_rule
    K = V = 128
    pool = torch.empty(140000, 1, K, V, device='cuda')   # 9 GB
    assert pool.numel() > 2 ** 31
    q, k, v, g, beta, s0 = (x if i == 5 else x[:, 0] for i, x in enumerate(R.delta_inputs(3, 1, 1, 1, K, V, BF16, seed=80)))
    slots = torch.tensor([139999, 0, 131073], device='cuda')
    pool[slots] = s0
    own = s0.clone()
    want = delta_rule.gated_delta_step(q, k, v, g, beta, own)
    got = delta_rule.gated_delta_step(q, k, v, g, beta, pool, slots=slots)
    assert torch.equal(got, want) and torch.equal(pool[slots], own)


def test_a_long_sequence_of_many_heads():
    """Against the last head alone, which may take other chunk sizes: two results of the same accuracy."""
    from blocks import delta_rule
    T, H, K, V = 70000, 256, 32, 128
    gen = torch.Generator(device='cuda').manual_seed(81)
    q, k = (torch.nn.functional.normalize(torch.randn(1, T, 1, K, generator=gen, device='cuda'), dim=-1).to(BF16) for _ in range(2))
    v = torch.randn(1, T, H, V, generator=gen, device='cuda', dtype=BF16)
    g, beta = -torch.rand(1, T, H, generator=gen, device='cuda'), torch.rand(1, T, H, generator=gen, device='cuda')
    assert v.numel() > 2 ** 31
    o, final = delta_rule.gated_delta_rule(q, k, v, g, beta)
    one, state = delta_rule.gated_delta_rule(q, k, v[:, :, -1:], g[:, :, -1:], beta[:, :, -1:])
    R.assert_close('final', final[:, -1:], state.cpu(), 2 * R.f32_atol(K + 128))
    half = torch.finfo(BF16).eps / 2
    R.assert_close('o', o[:, :, -1:], one.cpu(), 2 * R.o_atol(BF16, K), more=half * one.double().cpu().abs())


def test_many_short_sequences():
    from blocks import delta_rule
    B, T, H, K, V = 1100000, 2, 8, 1, 128
    gen = torch.Generator(device='cuda').manual_seed(82)
    q, k = (torch.randn(B, T, 1, K, generator=gen, device='cuda', dtype=BF16).clamp(-1, 1) for _ in range(2))
    v = torch.randn(B, T, H, V, generator=gen, device='cuda', dtype=BF16)
    g, beta = -torch.rand(B, T, H, generator=gen, device='cuda'), torch.rand(B, T, H, generator=gen, device='cuda')
    assert v.numel() > 2 ** 31
    ins = [x.requires_grad_() for x in (q, k, v, g, beta)]
    o, final = delta_rule.gated_delta_rule(*ins)
    do = torch.ones(1, dtype=BF16, device='cuda').expand(o.shape)
    got = torch.autograd.grad(o, ins, do)
    last = [x.detach()[-5:].requires_grad_() for x in ins]
    lo, lf = delta_rule.gated_delta_rule(*last)
    want = torch.autograd.grad(lo, last, do[-5:])
    assert torch.equal(o[-5:], lo) and torch.equal(final[-5:], lf)
    assert all(torch.equal(a[-5:], b) for a, b in zip(got, want))


def test_a_unit_of_many_rows():
    """y against the last rows alone, bit for bit (a row's sums do not depend on the others); dx too."""
    from blocks import gated_unit
    M, D, F = 2100000, 16, 1032
    gen = torch.Generator(device='cuda').manual_seed(83)
    x = torch.randn(M, D, generator=gen, device='cuda', dtype=BF16).requires_grad_()
    wg, wu = (torch.randn(D, F, generator=gen, device='cuda', dtype=BF16) / 4 for _ in range(2))
    assert M * F > 2 ** 31
    y = gated_unit.gated_unit(x, wg, wu)
    dy = torch.randn(1, F, generator=gen, device='cuda', dtype=BF16).expand(M, F)
    (dx,) = torch.autograd.grad(y, x, dy)
    last = x.detach()[-300:].requires_grad_()
    ly = gated_unit.gated_unit(last, wg, wu)
    (ldx,) = torch.autograd.grad(ly, last, dy[-300:])
    assert torch.equal(y[-300:], ly) and torch.equal(dx[-300:], ldx)
