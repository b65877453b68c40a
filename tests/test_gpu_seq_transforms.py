"""The sequence-layer operators under PyTorch's transformations, and on views that PyTorch evaluates late."""
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu


def _calls():
    """Each operator with gradients: its arguments and a call of them with one result."""
    from blocks.delta_rule import gated_delta_rule
    from blocks.dropout import dropout
    from blocks.gated_unit import gated_unit
    rule = R.delta_inputs(2, 40, 1, 2, 16, 24, torch.float32, seed=121)
    gen = torch.Generator().manual_seed(122)
    x, w, u, r = (torch.randn(s, generator=gen).cuda() for s in ((50, 16), (16, 24), (16, 24), (50, 16)))
    return {'rule': (rule, lambda *a: gated_delta_rule(*a[:5], initial_state=a[5])[0]), 'unit': ([x, w, u], gated_unit),
            'dropout': ([x, r], lambda a, b: dropout(a, 0.5, 3, residual=b))}


@pytest.mark.parametrize('name', ['rule', 'unit', 'dropout'])
def test_forward_mode_over_a_backward_pass_is_refused(name):
    import torch.autograd.forward_ad as fw
    args, call = _calls()[name]
    leaves = [t.requires_grad_() for t in args]
    y = call(*leaves)
    with fw.dual_level():
        dy = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize('name', ['rule', 'unit', 'dropout'])
def test_views_with_the_sign_turned_are_read_with_it(name):
    """The imaginary part of a conjugate is a view whose values PyTorch negates as they are read."""
    args, call = _calls()[name]
    dy = torch.randn_like(call(*args))
    want = torch.autograd.grad(call(*(t.requires_grad_() for t in args)), args, dy)
    y = call(*args).detach()
    turned = [torch._neg_view(-t.detach()) for t in args]
    assert all(t.is_neg() for t in turned)
    assert torch.equal(call(*turned), y)
    leaves = [(-t.detach()).requires_grad_() for t in args]
    out = call(*(torch._neg_view(t) for t in leaves))
    assert torch.equal(out.detach(), y)
    got = torch.autograd.grad(out, leaves, torch._neg_view(-dy))
    assert all(torch.equal(-a, b) for a, b in zip(got, want))
    z = torch.complex(torch.zeros_like(args[0].detach()), -args[0].detach()).conj().imag   # as programs come by them
    assert z.is_neg() and torch.equal(call(z, *args[1:]).detach(), y)


def test_single_tokens_with_the_sign_turned():
    from blocks.delta_rule import gated_delta_step
    q, k, v, g, beta, s0 = R.delta_inputs(3, 1, 1, 2, 16, 24, torch.float32, seed=123)
    args = [t[:, 0].contiguous() for t in (q, k, v, g, beta)]
    state = s0.clone()
    want = gated_delta_step(*args, state)
    again = s0.clone()
    assert torch.equal(gated_delta_step(*(torch._neg_view(-t) for t in args), again), want) and torch.equal(again, state)
    turned = torch._neg_view(-s0)
    with pytest.raises(ValueError, match='state'):
        gated_delta_step(*args, turned)
