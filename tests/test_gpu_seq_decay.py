"""The gated delta rule (blocks/delta_rule.py) where all rows decay strongly: gradients that are small themselves."""
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('T', [5, 32, 64, 130])
@pytest.mark.parametrize('decay', [-8.0, -12.0, -16.0])
def test_gradients_of_small_decays(decay, T, dtype):
    """Each value of dg has the factor exp(g), so the tensor's own root mean square, which the tolerance counts in, is as small.
    (The initial state's gradient is not compared: its factor exp(g T) is below the range of float32.)"""
    from blocks.delta_rule import gated_delta_rule
    K = V = 32
    ins = R.delta_inputs(2, T, 1, 2, K, V, dtype, seed=101)
    ins[3].fill_(decay)
    gen = torch.Generator(device='cuda').manual_seed(102)
    do = torch.randn(ins[2].shape, generator=gen, device='cuda').to(dtype)
    leaves = [x.requires_grad_() for x in ins[:5]]
    o, _ = gated_delta_rule(*leaves, initial_state=ins[5])
    got = torch.autograd.grad(o, leaves, do)
    ref = [x.detach().cpu().double().requires_grad_() for x in leaves]
    wo, _ = R.delta_rule(*ref, initial=ins[5].cpu())
    want = torch.autograd.grad(wo, ref, do.cpu().double())
    for n, a, b in zip(('q', 'k', 'v', 'g', 'beta'), got, want):
        R.assert_close('d' + n, a, b, R.grad_atol(a.dtype, K, V))
