"""The gated unit (blocks/gated_unit.py) on an MI355X against the formula in float64."""
import math

import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope='module')
def unit():
    from blocks.gated_unit import gated_unit
    return gated_unit


def _inputs(M, D, F, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * f).to(dtype).cuda()
            for s, f in (((M, D), 1.0), ((D, F), D ** -0.5), ((D, F), D ** -0.5), ((M, F), 1.0))]


def _check(unit, x, wg, wu, dy, act):
    dtype, D = x.dtype, x.size(-1)
    y0 = unit(x, wg, wu, activation=act)
    ref = [t.detach().cpu().double().requires_grad_() for t in (x, wg, wu)]
    want = R.gated_unit(*ref, act)
    R.assert_close('y', y0, want.detach(), R.unit_atol(D))
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    y = unit(*leaves, activation=act)
    assert torch.equal(y.detach(), y0)
    got = torch.autograd.grad(y, leaves, dy)
    wants = torch.autograd.grad(want, ref, dy.cpu().double())
    for n, a, b, (more, atol) in zip(('dx', 'dwg', 'dwu'), got, wants, R.unit_grad_bounds(x, wg, wu, dy, act)):
        assert a.dtype == dtype
        R.assert_close(n, a, b, atol, more)


SHAPES = [(1, 1, 1), (1, 8, 8), (3, 7, 5), (5, 64, 128), (17, 33, 65), (64, 64, 64), (65, 130, 72), (200, 96, 264), (130, 257, 129),
          (1, 1000, 300), (16, 520, 1000), (33, 72, 2000)]


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', SHAPES)
def test_values_and_gradients(unit, shape, dtype):
    x, wg, wu, dy = _inputs(*shape, dtype, seed=1)
    _check(unit, x, wg, wu, dy, 'silu')


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('act', ['gelu', 'sigmoid'])
def test_activations(unit, act, dtype):
    x, wg, wu, dy = _inputs(70, 40, 50, dtype, seed=2)
    _check(unit, x * 3, wg, wu, dy, act)


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('shape', [(2300, 320, 2052), (4100, 136, 1100)])
def test_large_tiles(unit, shape, dtype):
    """Sizes at which every product takes the large tiles in some direction, with ragged edges."""
    x, wg, wu, dy = _inputs(*shape, dtype, seed=3)
    _check(unit, x, wg, wu, dy, 'silu')


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_strides_and_alignment(unit, dtype):
    x, wg, wu, dy = _inputs(48, 40, 24, dtype, seed=4)
    wide = torch.zeros(48, 57, dtype=dtype, device='cuda')
    wide[:, 1:41] = x
    both = torch.cat([wg, wu], 1)
    for a, b, c in ((x.t().contiguous().t(), wg, wu), (wide[:, 1:41], wg, wu), (x, both[:, :24], both[:, 24:]),
                    (x, wg.t().contiguous().t(), wu), (x, wg, both[:, 24:])):
        _check(unit, a, b, c, dy, 'silu')
    _check(unit, x, wg, wu, dy.t().contiguous().t(), 'silu')
    _check(unit, x, wg, wu, dy[:1].expand(48, 24), 'silu')


def test_leading_axes_and_empty(unit):
    x, wg, wu, dy = _inputs(24, 16, 8, BF16, seed=5)
    y = unit(x.view(2, 3, 4, 16), wg, wu)
    assert y.shape == (2, 3, 4, 8) and torch.equal(y.view(24, 8), unit(x, wg, wu))
    assert torch.equal(unit(x[0], wg, wu), unit(x[:1], wg, wu)[0])
    leaves = [t.requires_grad_() for t in (x[:0].detach(), wg, wu)]
    y = unit(*leaves)
    assert y.shape == (0, 8)
    dx, dwg, dwu = torch.autograd.grad(y.sum(), leaves)
    assert dx.shape == (0, 16) and (dwg == 0).all() and (dwu == 0).all()


def test_only_the_gradients_that_are_wanted(unit):
    x, wg, wu, dy = _inputs(40, 32, 24, FP32, seed=6)
    a = [t.detach().requires_grad_() for t in (x, wg, wu)]
    full = torch.autograd.grad(unit(*a), a, dy)
    for i in range(3):
        b = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, wg, wu))]
        assert torch.equal(torch.autograd.grad(unit(*b), b[i], dy)[0], full[i])


def test_a_shared_weight_gets_both_gradients(unit):
    x, wg, _, dy = _inputs(40, 32, 24, FP32, seed=7)
    w = wg.detach().requires_grad_()
    (d,) = torch.autograd.grad(unit(x, w, w), w, dy)
    r = wg.detach().cpu().double().requires_grad_()
    (want,) = torch.autograd.grad(R.gated_unit(x.cpu(), r, r, 'silu'), r, dy.cpu().double())
    bounds = R.unit_grad_bounds(x, wg, wg, dy, 'silu')[1:]
    R.assert_close('dw', d, want, 2 * bounds[0][1], bounds[0][0] + bounds[1][0])


def test_not_finite_rows_stay_rows(unit):
    x, wg, wu, dy = _inputs(100, 72, 56, BF16, seed=8)
    clean = unit(x, wg, wu)
    x[17, 3] = math.nan
    y = unit(x, wg, wu)
    assert torch.isnan(y[17]).all()
    keep = torch.arange(100) != 17
    assert torch.equal(y[keep], clean[keep])


def test_gradients_against_differences(unit):
    """L is a sum of ~2000 f32 terms (error ~1e-5), 2h is at least 0.02 of the inputs' size: 1 % of the gradient's size is allowed."""
    x, wg, wu, dy = _inputs(60, 40, 30, FP32, seed=9)
    ins = [x, wg, wu]
    leaves = [t.detach().requires_grad_() for t in ins]
    grads = torch.autograd.grad(unit(*leaves), leaves, dy)
    for i in range(3):
        d = grads[i] / grads[i].norm()
        h = 1e-2 * float(ins[i].norm()) / 10
        up, dn = ([t + s * h * d if j == i else t for j, t in enumerate(ins)] for s in (1, -1))
        slope = float(((unit(*up) - unit(*dn)).double() * dy).sum()) / (2 * h)
        assert abs(slope - float(grads[i].norm())) <= 0.01 * float(grads[i].norm())


def test_captured_training_step(unit):
    x, wg, wu, dy = _inputs(100, 72, 90, BF16, seed=10)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]

    def step():
        y = unit(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            x.mul_(-0.75)
        graph.replay()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', [(1024, 40, 72), (5000, 64, 96), (33001, 24, 33), (9999, 300, 260)])
def test_many_rows_of_a_narrow_layer(unit, shape, dtype):
    """The weights' gradients summed in parts: few tiles, a long sum, its parts not of one length."""
    M, D, F = shape
    x, wg, wu, dy = _inputs(M, D, F, dtype, seed=31)
    _check(unit, x, wg, wu, dy, 'silu')
