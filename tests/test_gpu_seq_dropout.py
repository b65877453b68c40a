"""Dropout (blocks/dropout.py) on an MI355X against Philox4x32-10 and the formula in float64."""
import math

import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ATOL = 2.0 ** -22   # two f32 roundings (the factor, the product) before the sum, and the sum's


@pytest.fixture(scope='module')
def drop():
    from blocks.dropout import dropout
    return dropout


def _x(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', [(1,), (7,), (8,), (9,), (3, 5, 11), (64, 257), (1000, 1000)])
@pytest.mark.parametrize('residual', [False, True])
def test_values_and_gradients(drop, shape, dtype, residual):
    x, dy = _x(shape, dtype, 1).requires_grad_(), _x(shape, dtype, 2)
    r = _x(shape, dtype, 3).requires_grad_() if residual else None
    seed, offset = 0x0123456789abcdef, (1 << 40) + 5
    y = drop(x, 0.3, seed, offset=offset, residual=r)
    want, _ = R.dropout(x.detach(), 0.3, seed, offset, r.detach() if residual else None)
    R.assert_close('y', y.detach(), want, ATOL)
    got = torch.autograd.grad(y, [x, r] if residual else [x], dy)
    R.assert_close('dx', got[0], R.dropout(dy, 0.3, seed, offset)[0], ATOL)
    if residual:
        assert torch.equal(got[1], dy)


@pytest.mark.parametrize('p', [0.0, 1e-6, 1.0 / 65536, 0.5, 1 - 1.0 / 65536, 1.0])
def test_edges_of_p(drop, p):
    x = _x((300, 301), FP32, 4)
    y = drop(x, p, 7)
    want, keep = R.dropout(x, p, 7)
    R.assert_close('y', y, want, ATOL)
    assert torch.equal(y.cpu() != 0, keep)
    if p in (0.0, 1e-6):
        assert torch.equal(y, x)


def test_dropped_elements_count_as_zero_whatever_they_hold(drop):
    x = torch.full((4096,), math.nan, device='cuda')
    r = torch.ones_like(x)
    y = drop(x, 0.5, 11, residual=r).cpu()
    _, keep = R.dropout(x, 0.5, 11)
    assert torch.isnan(y[keep]).all() and (y[~keep] == 1).all()


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_unaligned_and_strided(drop, dtype):
    base = _x((70, 34), dtype, 5)
    for x in (base.flatten()[1:], base[:, 1:], base.t(), base[:, ::2]):
        R.assert_close('y', drop(x, 0.4, 3), R.dropout(x.contiguous(), 0.4, 3)[0], ATOL)


def test_empty(drop):
    x = torch.empty(0, 5, device='cuda', requires_grad=True)
    y = drop(x, 0.5, 1, residual=torch.empty(0, 5, device='cuda'))
    assert y.shape == (0, 5) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 5)


def test_counters_past_32_bits(drop):
    """Elements from 2^35 on would have counters from 2^32 on; the high word of the counter is checked by an offset instead, whose
    two words sit next to it, and by seeds that differ in their high words only."""
    x = torch.ones(4096, device='cuda')
    for seed, offset in ((5, 0), (5 + (1 << 32), 0), (5, 1 << 32), (5, 1), (-1, -1)):
        want, _ = R.dropout(x, 0.5, seed & (2 ** 64 - 1), offset & (2 ** 64 - 1))
        R.assert_close('y', drop(x, 0.5, seed, offset=offset), want, ATOL)


def test_kept_share(drop):
    """Of n = 4e6 fair draws the share kept differs from P(keep) by more than 5 sqrt(pq / n) once in a million seeds."""
    for p in (0.1, 0.5):
        n = 4_000_000
        kept = float((drop(torch.ones(n, device='cuda'), p, 12345) != 0).double().mean())
        assert abs(kept - (1 - p)) <= 5 * math.sqrt(p * (1 - p) / n) + 1 / 131072


def test_seed_on_the_device_and_captured(drop):
    x = _x((50, 99), BF16, 6).requires_grad_()
    seed = torch.tensor([41], device='cuda')
    assert torch.equal(drop(x, 0.5, seed), drop(x, 0.5, 41))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(drop(x, 0.5, seed, offset=3).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x, 0.5, seed, offset=3)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    for s in (1, 2, 1 << 40):
        seed.fill_(s)
        graph.replay()
        torch.cuda.synchronize()
        want, keep = R.dropout(x.detach(), 0.5, s, 3)
        R.assert_close('y', y.detach(), want, ATOL)
        assert torch.equal(dx.cpu() != 0, keep)


def test_editing_the_seed_between_the_passes_is_an_error(drop):
    x = _x((8,), FP32).requires_grad_()
    seed = torch.tensor([1], device='cuda')
    y = drop(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
