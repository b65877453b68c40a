"""Sequences of at most 32 rows of blocks/delta_rule.py, which take one kernel each way, against the float64 recurrence."""
import math

import pytest
import torch

import seq_reference as R
from test_gpu_seq_delta import BF16, FP16, FP32, _check, _check_grads, _grads

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def rule():
    from blocks import delta_rule
    return delta_rule


# B, T, Hk, Hv, K, V: every size of head, one row to 32, columns in several passes, odd sizes, shared query/key heads
SHAPES = [(1, 1, 1, 1, 1, 1), (3, 2, 1, 2, 16, 16), (2, 31, 2, 2, 24, 40), (5, 32, 2, 4, 32, 64), (1, 17, 1, 3, 33, 17),
          (4, 32, 2, 2, 64, 64), (2, 16, 2, 4, 64, 130), (1, 30, 1, 1, 100, 72), (2, 32, 1, 2, 128, 128), (1, 5, 1, 1, 127, 250),
          (700, 3, 1, 2, 8, 20)]


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', SHAPES)
def test_values_and_gradients(rule, shape, dtype):
    B, T, Hk, Hv, K, V = shape
    _check_grads(rule, R.delta_inputs(B, T, Hk, Hv, K, V, dtype, seed=41), dtype)


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_strided_and_unaligned_inputs(rule, dtype):
    B, T, H, K, V = 3, 20, 2, 24, 40
    gen = torch.Generator(device='cuda').manual_seed(42)
    w = torch.randn(T, B, H * (2 * K + V) + 3, generator=gen, device='cuda').to(dtype).transpose(0, 1)
    part = w[:, :, 1:1 + H * (2 * K + V)].unflatten(-1, (H, 2 * K + V))
    q, k, v = part[..., :K] * 0.2, part[..., K:2 * K] * 0.2, part[..., 2 * K:]
    wide = torch.empty(B, T, H, 2 * K + V + 1, dtype=dtype, device='cuda')
    wide[..., 1:K + 1], wide[..., K + 1:2 * K + 1] = q, k
    q, k = wide[..., 1:K + 1], wide[..., K + 1:2 * K + 1]
    _, _, _, g, beta, s0 = R.delta_inputs(B, T, H, H, K, V, dtype, seed=43)
    g, beta = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (g, beta))
    _check_grads(rule, (q, k, v, g, beta, s0), dtype)


def test_rows_far_apart_and_the_same_row_again(rule):
    """Strides past what the one kernel's 32-bit offsets reach (rows 2^25 values apart), and of zero."""
    q, k, v, g, beta, s0 = R.delta_inputs(1, 3, 1, 1, 16, 16, BF16, seed=44)
    far = torch.empty(2 * 2 ** 25 + 16, dtype=BF16, device='cuda').as_strided((1, 3, 1, 16), (16, 2 ** 25, 16, 1))
    near = torch.empty(2 * (2 ** 25 - 8) + 16, dtype=BF16, device='cuda').as_strided((1, 3, 1, 16), (16, 2 ** 25 - 8, 16, 1))
    far.copy_(v)
    near.copy_(v)
    for x in (far, near):
        _check(rule, (q, k, x, g, beta, s0), 16, BF16)
        _check(rule, (x * 0.2, k, v, g, beta, s0), 16, BF16)
    _check(rule, (q, k[:, :1].expand(1, 3, 1, 16), v[:, :1].expand(1, 3, 1, 16), g, beta, s0), 16, BF16)


def test_strong_decay_and_resets(rule):
    q, k, v, g, beta, s0 = R.delta_inputs(2, 32, 1, 2, 32, 32, FP32, seed=45)
    g[:, 4:30] -= 30.0
    g[:, 7] = -math.inf
    g[:, 20, 1] = -math.inf
    _check(rule, (q, k, v, g, beta, s0), 32, FP32)
    leaves = [x.requires_grad_() for x in (q, k, v, g, beta, s0)]
    o, final = rule.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    grads = torch.autograd.grad([o, final], leaves, [torch.ones_like(o), torch.ones_like(final)])
    assert all(torch.isfinite(x).all() for x in grads) and (grads[3][:, 7] == 0).all()


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('which, value', [('k', math.nan), ('k', math.inf), ('g', math.nan), ('beta', math.nan), ('q', math.nan),
                                          ('v', math.inf)])
def test_what_is_not_finite_changes_nothing_before_it(rule, which, value, dtype):
    ins = R.delta_inputs(2, 29, 1, 2, 16, 20, dtype, seed=46)
    clean = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
    x = ins['qkvg'.index(which) if which != 'beta' else 4]
    x[(0, 13, 0) if x.dim() == 3 else (0, 13, 0, 2)] = value
    o, final = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
    heads = slice(None) if which in 'qk' else slice(0, 1)
    cols = slice(2, 3) if which == 'v' else slice(None)
    rows = slice(13, 14) if which == 'q' else slice(13, None)
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, rows, heads, cols] = True
    assert torch.equal(torch.isnan(o), hit) and torch.equal(o[~hit], clean[0][~hit])
    gone = torch.zeros_like(final, dtype=torch.bool)
    if which != 'q':
        gone[0, heads, :, cols] = True
    assert torch.equal(torch.isnan(final), gone) and torch.equal(final[~gone], clean[1][~gone])


def test_every_other_column_is_right_beside_one_that_is_not_finite(rule):
    """A column with an infinity beside finite ones in the same wave: theirs come out as the recurrence has them."""
    for T in (24, 90):
        q, k, v, g, beta, s0 = R.delta_inputs(1, T, 1, 1, 32, 16, FP32, seed=47)
        wo, wf = R.delta_rule(*(x.cpu() for x in (q, k, v, g, beta)), initial=s0.cpu())
        v[0, 5, 0, 3] = math.inf
        o, final = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
        others = [c for c in range(16) if c != 3]
        R.assert_close('o', o[..., others], wo[..., others], R.o_atol(FP32, 32))
        R.assert_close('final', final[..., others], wf[..., others], R.f32_atol(32 + 128))


def test_without_an_initial_state_and_its_gradient(rule):
    q, k, v, g, beta, _ = R.delta_inputs(2, 32, 2, 4, 64, 70, FP32, seed=48)
    leaves = [x.requires_grad_() for x in (q, k, v, g, beta)]
    o, final = rule.gated_delta_rule(*leaves)
    got = torch.autograd.grad(o.sum(), leaves)   # no gradient of the final state either
    ref = [x.detach().cpu().double().requires_grad_() for x in leaves]
    want = torch.autograd.grad(R.delta_rule(*ref)[0].sum(), ref)
    for n, a, b in zip('qkvgb', got, want):
        R.assert_close('d' + n, a, b, R.grad_atol(FP32, 64, 70))


def test_gradients_against_differences(rule):
    """As for long sequences: L is a sum of ~1e4 f32 terms of size ~1, 2 % of the gradient's size is allowed."""
    ins = R.delta_inputs(4, 32, 1, 2, 32, 24, FP32, seed=49)
    gen = torch.Generator(device='cuda').manual_seed(6)
    do = torch.randn(ins[2].shape, generator=gen, device='cuda')
    df = torch.randn(ins[5].shape, generator=gen, device='cuda')
    grads = _grads(rule, ins, do, df)[4]

    def loss(xs):
        o, f = rule.gated_delta_rule(*xs[:5], initial_state=xs[5])
        return float((o.double() * do).sum() + (f.double() * df).sum())

    for i, d in enumerate(grads):
        d, size = d / d.norm(), float(d.norm())
        h = 1e-2 * float(ins[i].norm()) / 10
        up = [x + h * d if j == i else x for j, x in enumerate(ins)]
        dn = [x - h * d if j == i else x for j, x in enumerate(ins)]
        assert abs((loss(up) - loss(dn)) / (2 * h) - size) <= 0.02 * size, i


def test_captured_training_step(rule):
    """Forward and backward in one graph, replayed on new values in the same places."""
    ins = [x.requires_grad_() for x in R.delta_inputs(6, 32, 1, 2, 32, 32, BF16, seed=50)]
    do = torch.randn_like(ins[2])

    def step():
        o, f = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
        return (o, f, *torch.autograd.grad([o, f], ins, [do, torch.ones_like(f)]))

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
            do.mul_(-0.5)
            ins[2].add_(0.25)
        graph.replay()
        got = [x.clone() for x in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i


def test_no_rows_and_no_sequences(rule):
    for B, T in ((0, 8), (3, 0)):
        ins = [x.requires_grad_() for x in R.delta_inputs(B, T, 1, 2, 16, 20, BF16, seed=51)]
        o, final = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
        assert o.shape == (B, T, 2, 20) and torch.equal(final, ins[5])
        grads = torch.autograd.grad([o, final], ins, [torch.ones_like(o), torch.ones_like(final)])
        assert torch.equal(grads[5], torch.ones_like(final)) and all(d.shape == x.shape for d, x in zip(grads, ins))


def test_a_graph_of_the_gradients_is_refused(rule):
    for T in (16, 80):
        ins = [x.requires_grad_() for x in R.delta_inputs(1, T, 1, 1, 16, 16, FP32, seed=52)]
        o, _ = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
        (d,) = torch.autograd.grad(o.sum(), ins[2], create_graph=True)
        with pytest.raises(RuntimeError):
            d.sum().backward()
