"""Many sequences and heads of blocks/delta_rule.py at once: the chunk sizes and column shares chosen for them, against the float64
recurrence."""
import pytest
import torch

import seq_reference as R
from test_gpu_seq_delta import BF16, FP16, FP32, _check, _check_grads

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def rule():
    from blocks import delta_rule
    return delta_rule


# B, T, Hk, Hv, K, V: from 288 to 640 tiles of 16 columns
SHAPES = [(24, 70, 2, 4, 32, 96), (9, 70, 4, 8, 128, 120), (20, 67, 4, 4, 60, 128), (40, 48, 2, 4, 64, 50), (9, 65, 4, 4, 40, 128)]


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', SHAPES)
def test_sequences(rule, shape, dtype):
    B, T, Hk, Hv, K, V = shape
    ins = R.delta_inputs(B, T, Hk, Hv, K, V, dtype, seed=61)
    with torch.no_grad():
        _check(rule, ins, K, dtype)
    _check_grads(rule, ins, dtype)


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('mean', [20, 45, 90])
def test_packed_sequences(rule, dtype, mean):
    n = 22
    lengths = torch.tensor([0, 1, 31, 32, 33, 63, 64, 65] + [1 + i * mean // 6 for i in range(n - 8)])
    lengths = lengths * mean * n // int(lengths.sum())
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), lengths.cumsum(0)]).int().cuda()
    ins = R.delta_inputs(1, int(offsets[-1]) + 5, 2, 4, 64, 100, dtype, seed=62, n=n)
    with torch.no_grad():
        _check(rule, ins, 64, dtype, offsets=offsets)
    _check_grads(rule, ins, dtype, offsets=offsets)
