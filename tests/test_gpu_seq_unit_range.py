"""The gated unit (blocks/gated_unit.py) over the range of its types: gradients of float16 outside the range in which float16 holds
the projections' own gradients, and values at the ends of float32."""
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

FP16, FP32 = torch.float16, torch.float32


@pytest.fixture(scope='module')
def unit():
    from blocks.gated_unit import gated_unit
    return gated_unit


def _gradients(unit, x, wg, wu, dy, act):
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(unit(*leaves, activation=act), leaves, dy)
    ref = [t.detach().cpu().double().requires_grad_() for t in (x, wg, wu)]
    return got, torch.autograd.grad(R.gated_unit(*ref, act), ref, dy.cpu().double())


def _check_fp16(unit, M, D, F, x_size, dy_size, act):
    """float16 operands and the projections' gradients are two bf16 pieces each: 2^-16 of a term is what the second one of a
    gradient is rounded by, as much is left out as the product of both second pieces; 2^-25 is half a step below the normal range.
    The rest is that of float32 sums."""
    gen = torch.Generator().manual_seed(111)
    x, wg, wu, dy = ((torch.randn(s, generator=gen) * f).to(FP16).cuda() for s, f in
                     (((M, D), x_size), ((D, F), D ** -0.5), ((D, F), D ** -0.5), ((M, F), dy_size)))
    got, want = _gradients(unit, x, wg, wu, dy, act)
    bounds = R.unit_grad_bounds(*(t.double() for t in (x, wg, wu, dy)), act)
    for n, a, b, (more, atol), terms in zip(('dx', 'dwg', 'dwu'), got, want, bounds, (2 * F, M, M)):
        assert a.dtype == FP16
        a, b = a.cpu(), b.clone()
        beyond, edge = b.abs() > 65520 * (1 + 2.0 ** -9), b.abs() > 65504 * (1 - 2.0 ** -9)   # no float16 has this value; may have none
        assert torch.equal(a[beyond], b[beyond].sign().half() * float('inf'))
        assert n != 'dx' or not edge.any()
        a[edge] = b[edge] = 0
        sizes = more / (torch.finfo(torch.float64).eps / 2 + terms * 2.0 ** -24)
        R.assert_close(n, a, b, atol, more + 2.0 ** -15 * sizes + 2.0 ** -25)


@pytest.mark.parametrize('act', ['silu', 'gelu', 'sigmoid'])
@pytest.mark.parametrize('dy_size', [1e-5, 1e-3, 30.0])
def test_gradients_of_fp16_small_and_large(unit, dy_size, act):
    _check_fp16(unit, 700, 72, 136, 1.0, dy_size, act)


def test_gradients_of_fp16_whose_parts_are_beyond_it(unit):
    """dy b act' is up to 1.4e5, dx below 35000; most of the weights' gradients are infinite in float16, as they should be."""
    _check_fp16(unit, 16, 1024, 64, 8.0, 4000.0, 'silu')


@pytest.mark.parametrize('shape', [(40, 33, 65), (2300, 320, 2052), (33001, 24, 33)])
def test_gradients_of_fp16_in_every_tile_and_in_parts(unit, shape):
    _check_fp16(unit, *shape, 1.0, 1e-4, 'silu')


def _fp32(M, D, F, x_size, w_size, dy_size):
    gen = torch.Generator().manual_seed(112)
    return [torch.randn(s, generator=gen) * f for s, f in (((M, D), x_size), ((D, F), w_size), ((D, F), w_size), ((M, F), dy_size))]


@pytest.mark.parametrize('M', [5, 100])
def test_the_largest_values_of_fp32(unit, M):
    """Those above the largest bf16 value (3.39e38) would be infinities as bf16; weights and dy are so small that all results are in
    range, with as much room below."""
    D, F = 24, 40
    x, wg, wu, dy = (t.cuda() for t in _fp32(M, D, F, 1.2e38, 1e-30, 1e-12))
    x.clamp_(-torch.finfo(FP32).max, torch.finfo(FP32).max)
    x[::2, 3], x[1::2, 5] = torch.finfo(FP32).max, -3.398e38
    y = unit(x, wg, wu)
    R.assert_close('y', y, R.gated_unit(x.cpu(), wg.cpu(), wu.cpu(), 'silu'), R.unit_atol(D))
    got, want = _gradients(unit, x, wg, wu, dy, 'silu')
    for n, a, b, (more, atol) in zip(('dx', 'dwg', 'dwu'), got, want, R.unit_grad_bounds(x, wg, wu, dy, 'silu')):
        R.assert_close(n, a, b, atol, more)


@pytest.mark.parametrize('M', [5, 100])
def test_an_infinity_of_fp32_counts_as_nan(unit, M):
    """Whichever kernel the number of rows leads to."""
    x, wg, wu, _ = (t.cuda() for t in _fp32(M, 24, 40, 1.0, 0.2, 1.0))
    clean = unit(x, wg, wu, activation='sigmoid')
    for value in (float('inf'), -float('inf')):
        for t, at, hit in ((x, (3, 7), (3, slice(None))), (wg, (23, 9), (slice(None), 9)), (wu, (0, 39), (slice(None), 39))):
            was = t[at].clone()
            t[at] = value
            y = unit(x, wg, wu, activation='sigmoid')
            t[at] = was
            gone = torch.zeros_like(y, dtype=torch.bool)
            gone[hit] = True
            assert torch.equal(torch.isnan(y), gone) and torch.equal(y[~gone], clean[~gone])
