"""What the sequence-layer operators refuse of PyTorch's transformations, which would otherwise lose their results without a word.
Without a GPU: these are refused before anything is computed."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def _calls():
    """Each operator's arguments, and a call of them."""
    from blocks.delta_rule import gated_delta_rule, gated_delta_step
    from blocks.dropout import dropout
    from blocks.gated_unit import gated_unit
    rule = [torch.randn(2, 5, 1, 8), torch.randn(2, 5, 1, 8), torch.randn(2, 5, 2, 4), torch.randn(2, 5, 2), torch.randn(2, 5, 2)]
    return {
        'rule': (rule + [torch.randn(2, 2, 8, 4)], lambda *a: gated_delta_rule(*a[:5], initial_state=a[5])),
        'step': ([x[:, 0] for x in rule] + [torch.randn(2, 2, 8, 4)], gated_delta_step),
        'unit': ([torch.randn(3, 4), torch.randn(4, 5), torch.randn(4, 5)], gated_unit),
        'dropout': ([torch.randn(3, 4), torch.randn(3, 4)], lambda x, r: dropout(x, 0.5, 1, residual=r)),
    }


ARGS = [('rule', i) for i in range(6)] + [('step', i) for i in range(6)] + [('unit', i) for i in range(3)] + [('dropout', i) for i in range(2)]


@pytest.mark.parametrize('name, which', ARGS)
@pytest.mark.parametrize('leaf', [False, True])
def test_forward_mode_is_refused(name, which, leaf):
    import torch.autograd.forward_ad as fw
    args, call = _calls()[name]
    if leaf:
        args[which].requires_grad_()
    with fw.dual_level():
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match='forward-mode'):
            call(*args)


@pytest.mark.parametrize('name', ['rule', 'step', 'unit', 'dropout'])
def test_tracing_is_refused(name):
    args, call = _calls()[name]
    with pytest.raises(RuntimeError, match='traced'):
        torch.jit.trace(call, tuple(args), check_trace=False)


@pytest.mark.parametrize('name, which', ARGS)
def test_tensors_without_memory_of_their_own_are_refused(name, which):
    args, call = _calls()[name]
    batched = list(args)
    batched[which] = torch.stack([args[which]] * 3)
    with pytest.raises(TypeError, match='memory of its own'):
        torch.func.vmap(call, in_dims=tuple(0 if i == which else None for i in range(len(args))))(*batched)
    sparse = list(args)
    sparse[which] = args[which].to_sparse()
    with pytest.raises(TypeError, match='memory of its own'):
        call(*sparse)
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = list(args)
        fake[which] = mode.from_tensor(args[which])
        with pytest.raises(TypeError, match='memory of its own'):
            call(*fake)
