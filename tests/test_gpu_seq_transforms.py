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
