"""The gated delta rule (blocks/delta_rule.py) on an MI355X against the token-by-token recurrence in float64."""
import math

import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope='module')
def rule():
    from blocks import delta_rule
    return delta_rule


def _check(rule, ins, K, dtype, **kw):
    q, k, v, g, beta, s0 = ins
    o, final = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0, **kw)
    ref = {n: (x.cpu() if isinstance(x, torch.Tensor) else x) for n, x in kw.items()}
    wo, wf = R.delta_rule(*(x.cpu() for x in (q, k, v, g, beta)), initial=None if s0 is None else s0.cpu(), **ref)
    assert o.dtype == dtype and final.dtype == torch.float32
    R.assert_close('final', final, wf, R.f32_atol(K + 128))
    R.assert_close('o', o, wo, R.o_atol(dtype, K))


# lengths around the 64-row chunk, odd and padded head sizes, shared query/key heads
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 1, 2, 16, 16), (1, 63, 2, 2, 24, 40), (2, 64, 1, 3, 32, 16), (1, 65, 2, 4, 33, 17),
          (1, 130, 1, 1, 64, 65), (2, 200, 2, 2, 100, 72), (1, 321, 1, 2, 128, 128), (3, 40, 2, 2, 7, 250)]


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', SHAPES)
def test_sequences(rule, shape, dtype):
    B, T, Hk, Hv, K, V = shape
    _check(rule, R.delta_inputs(B, T, Hk, Hv, K, V, dtype, seed=1), K, dtype)


@pytest.mark.parametrize('T', [0, 5])
def test_no_initial_state_and_no_rows(rule, T):
    q, k, v, g, beta, s0 = R.delta_inputs(2, T, 2, 2, 16, 16, FP32)
    _check(rule, (q, k, v, g, beta, None), 16, FP32)
    o, final = rule.gated_delta_rule(q[:0], k[:0], v[:0], g[:0], beta[:0])
    assert o.shape == (0, T, 2, 16) and final.shape == (0, 2, 16, 16)
    if T == 0:
        _, final = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
        assert torch.equal(final, s0)


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('wide', [torch.int32, torch.int64])
def test_packed_sequences(rule, dtype, wide):
    """Empty sequences first, in the middle and last; lengths that end in a chunk, on its edge, and one row past it."""
    off = torch.tensor([0, 0, 1, 65, 65, 193, 194, 260, 260], dtype=wide, device='cuda')
    ins = R.delta_inputs(1, 260, 2, 4, 40, 24, dtype, seed=2, n=8)
    _check(rule, ins, 40, dtype, offsets=off)


def test_rows_outside_the_packed_sequences_are_zero(rule):
    off = torch.tensor([5, 70, 90], dtype=torch.int32, device='cuda')
    q, k, v, g, beta, s0 = R.delta_inputs(1, 200, 1, 2, 16, 24, BF16, seed=3, n=2)
    for t in (q, k, v, g, beta):   # whatever those rows hold
        t[:, :5] = math.nan
        t[:, 90:] = math.inf
    o, final = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0, offsets=off)
    assert torch.equal(o[:, :5], torch.zeros_like(o[:, :5])) and torch.equal(o[:, 90:], torch.zeros_like(o[:, 90:]))
    wo, wf = R.delta_rule(*(x[:, :90].cpu() for x in (q, k, v, g, beta)), initial=s0.cpu(), offsets=off.cpu())
    R.assert_close('final', final, wf, R.f32_atol(16 + 128))
    R.assert_close('o', o[:, 5:90], wo[:, 5:90], R.o_atol(BF16, 16))


def test_offsets_out_of_range_are_taken_as_the_nearest_inside(rule):
    q, k, v, g, beta, s0 = R.delta_inputs(1, 100, 1, 1, 16, 16, FP32, seed=4, n=2)
    got = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0,
                                offsets=torch.tensor([-7, 40, 1 << 30], dtype=torch.int32, device='cuda'))
    want = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0,
                                 offsets=torch.tensor([0, 40, 100], dtype=torch.int64, device='cuda'))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_strided_and_unaligned_inputs(rule, dtype):
    """Slices of one fused projection, a batch stride that is not the time axis', unaligned first values."""
    B, T, H, K, V = 2, 70, 2, 24, 40
    gen = torch.Generator(device='cuda').manual_seed(5)
    w = torch.randn(T, B, H * (2 * K + V) + 3, generator=gen, device='cuda').to(dtype).transpose(0, 1)
    part = w[:, :, 1:1 + H * (2 * K + V)].unflatten(-1, (H, 2 * K + V))
    q, k, v = part[..., :K] * 0.2, part[..., K:2 * K] * 0.2, part[..., 2 * K:]
    wide = torch.empty(B, T, H, 2 * K + V + 1, dtype=dtype, device='cuda')
    wide[..., 1:K + 1], wide[..., K + 1:2 * K + 1] = q, k
    q, k = wide[..., 1:K + 1], wide[..., K + 1:2 * K + 1]
    assert not (q.is_contiguous() or v.is_contiguous())
    _, _, _, g, beta, s0 = R.delta_inputs(B, T, H, H, K, V, dtype, seed=6)
    g, beta = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (g, beta))
    _check(rule, (q, k, v, g, beta, s0), K, dtype)
    _check(rule, (q.transpose(2, 3).contiguous().transpose(2, 3), k, v, g, beta, s0), K, dtype)   # last axis strided


def test_strong_decay_and_resets(rule):
    """Sums of g in the thousands, and -inf, which starts the state afresh: exp of differences, never of the sums."""
    q, k, v, g, beta, s0 = R.delta_inputs(1, 150, 1, 2, 32, 32, FP32, seed=7)
    g[:, 10:140] -= 30.0
    g[:, 20] = -math.inf
    g[:, 100, 1] = -math.inf
    _check(rule, (q, k, v, g, beta, s0), 32, FP32)


def test_zero_strengths_and_repeated_keys(rule):
    q, k, v, g, beta, s0 = R.delta_inputs(1, 130, 1, 1, 16, 16, FP32, seed=8)
    beta[:, 3::7] = 0.0
    k[:, 64:96] = k[:, 64:65]
    g[:, 64:96] = 0.0
    _check(rule, (q, k, v, g, beta, s0), 16, FP32)


def test_a_nan_stays_in_its_sequence_and_head(rule):
    q, k, v, g, beta, s0 = R.delta_inputs(2, 70, 2, 2, 16, 16, FP32, seed=9)
    v[0, 30, 1, 3] = math.nan
    o, final = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    bad = torch.isnan(final)
    assert bad[0, 1, :, 3].all() and int(bad.sum()) == 16
    assert not torch.isnan(o[0, :30]).any() and torch.isnan(o[0, 30:, 1, 3]).all() and not torch.isnan(o[1]).any()


@pytest.mark.parametrize('which, value', [('k', math.nan), ('k', math.inf), ('g', math.nan), ('beta', math.nan), ('q', math.nan),
                                          ('v', math.inf)])
def test_what_is_not_finite_changes_nothing_before_it(rule, which, value):
    ins = R.delta_inputs(2, 130, 1, 2, 16, 20, BF16, seed=17)
    clean = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
    x = ins['qkvg'.index(which) if which != 'beta' else 4]
    x[(0, 70, 0) if x.dim() == 3 else (0, 70, 0, 2)] = value
    o, final = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
    heads = slice(None) if which in 'qk' else slice(0, 1)
    cols = slice(2, 3) if which == 'v' else slice(None)
    rows = slice(70, 71) if which == 'q' else slice(70, None)
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, rows, heads, cols] = True
    assert torch.equal(torch.isnan(o), hit) and torch.equal(o[~hit], clean[0][~hit])
    gone = torch.zeros_like(final, dtype=torch.bool)
    if which != 'q':
        gone[0, heads, :, cols] = True
    assert torch.equal(torch.isnan(final), gone) and torch.equal(final[~gone], clean[1][~gone])


def test_a_sequence_in_two_calls_is_the_sequence_in_one(rule):
    q, k, v, g, beta, s0 = R.delta_inputs(2, 192, 2, 2, 32, 48, FP32, seed=10)
    whole = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    a = rule.gated_delta_rule(*(x[:, :128] for x in (q, k, v, g, beta)), initial_state=s0)
    b = rule.gated_delta_rule(*(x[:, 128:] for x in (q, k, v, g, beta)), initial_state=a[1])
    assert torch.equal(torch.cat([a[0], b[0]], 1), whole[0]) and torch.equal(b[1], whole[1])   # cut on a chunk's edge


# ---------------------------------------------------------------------------------------------------- gradients

NAMES = ('q', 'k', 'v', 'g', 'beta', 'initial')


def _grads(rule, ins, do, dfinal, **kw):
    """Gradients of <o, do> + <final, dfinal> from the kernels and from the float64 recurrence."""
    leaves = [x.detach().requires_grad_() for x in ins]
    o, final = rule.gated_delta_rule(*leaves[:5], initial_state=leaves[5], **kw)
    got = torch.autograd.grad([o, final], leaves, [do, dfinal])
    ref = [x.detach().cpu().double().requires_grad_() for x in ins]
    wo, wf = R.delta_rule(*ref[:5], initial=ref[5], **{n: x.cpu() for n, x in kw.items()})
    want = torch.autograd.grad([wo, wf], ref, [do.cpu().double(), dfinal.cpu().double()], allow_unused=True)
    return o, final, wo, wf, got, [torch.zeros_like(r) if w is None else w for r, w in zip(ref, want)]


def _check_grads(rule, ins, dtype, **kw):
    gen = torch.Generator(device='cuda').manual_seed(99)
    K, V = ins[5].shape[2:]
    do = torch.randn(ins[2].shape, generator=gen, device='cuda').to(dtype)
    dfinal = torch.randn(ins[5].shape, generator=gen, device='cuda')
    o, final, wo, wf, got, want = _grads(rule, ins, do, dfinal, **kw)
    R.assert_close('o', o.detach(), wo.detach(), R.o_atol(dtype, K))
    R.assert_close('final', final.detach(), wf.detach(), R.f32_atol(K + 128))
    for n, a, b, leaf in zip(NAMES, got, want, ins):
        assert a.dtype == leaf.dtype and a.shape == leaf.shape
        R.assert_close('d' + n, a, b, R.grad_atol(a.dtype, K, V))


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', SHAPES)
def test_gradients(rule, shape, dtype):
    B, T, Hk, Hv, K, V = shape
    _check_grads(rule, R.delta_inputs(B, T, Hk, Hv, K, V, dtype, seed=21), dtype)


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_gradients_of_packed_sequences(rule, dtype):
    off = torch.tensor([0, 0, 1, 65, 65, 193, 194, 260, 260], dtype=torch.int32, device='cuda')
    _check_grads(rule, R.delta_inputs(1, 260, 2, 4, 40, 24, dtype, seed=22, n=8), dtype, offsets=off)


def test_rows_outside_the_packed_sequences_get_zero_gradients(rule):
    off = torch.tensor([5, 70, 90], dtype=torch.int32, device='cuda')
    ins = R.delta_inputs(1, 200, 1, 2, 16, 24, BF16, seed=23, n=2)
    leaves = [x.requires_grad_() for x in ins]
    o, final = rule.gated_delta_rule(*leaves[:5], initial_state=leaves[5], offsets=off)
    do = torch.full_like(o, math.nan)
    do[:, 5:90] = 1.0
    for n, d in zip(NAMES[:5], torch.autograd.grad([o, final], leaves, [do, torch.ones_like(final)])):
        assert torch.isfinite(d).all(), n
        assert (d[:, :5] == 0).all() and (d[:, 90:] == 0).all() and (d[:, 5:90] != 0).any(), n


def test_gradients_with_strong_decay_and_resets(rule):
    ins = R.delta_inputs(1, 150, 1, 2, 32, 32, FP32, seed=24)
    ins[3][:, 10:140] -= 30.0
    _check_grads(rule, ins, FP32)
    ins[3][:, 20] = -math.inf
    leaves = [x.requires_grad_() for x in ins]
    o, final = rule.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    grads = torch.autograd.grad([o, final], leaves, [torch.ones_like(o), torch.ones_like(final)])
    assert all(torch.isfinite(x).all() for x in grads) and (grads[3][:, 20] == 0).all()


def test_gradients_of_strided_inputs_and_without_an_initial_state(rule):
    q, k, v, g, beta, _ = R.delta_inputs(2, 70, 2, 2, 24, 40, FP32, seed=25)
    fused = torch.cat([q, k, v], -1).requires_grad_()
    o, final = rule.gated_delta_rule(fused[..., :24], fused[..., 24:48], fused[..., 48:], g, beta)
    (d,) = torch.autograd.grad(o.sum() + final.sum(), fused)
    ref = fused.detach().cpu().double().requires_grad_()
    wo, wf = R.delta_rule(ref[..., :24], ref[..., 24:48], ref[..., 48:], g.cpu(), beta.cpu())
    (w,) = torch.autograd.grad(wo.sum() + wf.sum(), ref)
    R.assert_close('d', d, w, R.grad_atol(FP32, 24, 40))


def test_gradients_against_differences(rule):
    """Along one direction: (L(x + h d) - L(x - h d)) / 2h.  L is a sum of ~1e4 f32 terms of size ~1 (error ~1e-4 in L, 1e-2
    after division by 2h = 0.02), the third derivative adds ~h^2 relative: 2 % of the gradient's size is allowed."""
    ins = R.delta_inputs(2, 100, 1, 2, 32, 24, FP32, seed=26)
    gen = torch.Generator(device='cuda').manual_seed(5)
    do = torch.randn(ins[2].shape, generator=gen, device='cuda')
    df = torch.randn(ins[5].shape, generator=gen, device='cuda')

    def loss(xs):
        o, f = rule.gated_delta_rule(*xs[:5], initial_state=xs[5])
        return float((o.double() * do).sum() + (f.double() * df).sum())

    leaves = [x.detach().requires_grad_() for x in ins]
    o, f = rule.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    grads = torch.autograd.grad([o, f], leaves, [do, df])
    for i, n in enumerate(NAMES):
        d = grads[i] / grads[i].norm()
        h = 1e-2 * float(ins[i].norm()) / 10
        up = [x + h * d if j == i else x for j, x in enumerate(ins)]
        dn = [x - h * d if j == i else x for j, x in enumerate(ins)]
        slope = (loss(up) - loss(dn)) / (2 * h)
        assert abs(slope - float(grads[i].norm())) <= 0.02 * float(grads[i].norm()), n


def test_gradients_twice_and_after_an_edit(rule):
    ins = [x.requires_grad_() for x in R.delta_inputs(1, 80, 1, 1, 16, 16, FP32, seed=27)]
    o, _ = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
    a = torch.autograd.grad(o.sum(), ins, retain_graph=True)
    b = torch.autograd.grad(o.sum(), ins)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    o, _ = rule.gated_delta_rule(*ins[:5], initial_state=ins[5])
    with torch.no_grad():
        ins[2].add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        o.sum().backward()


def test_captured_training_step(rule):
    """Forward and backward in one graph, replayed on new values in the same places."""
    ins = [x.requires_grad_() for x in R.delta_inputs(2, 100, 1, 2, 32, 32, BF16, seed=28)]
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


# ------------------------------------------------------------------------------------------------ single tokens

# the last two: enough heads for whole rows of columns in a workgroup
STEPS = [(1, 1, 1, 1, 1), (3, 2, 4, 32, 32), (2, 1, 3, 33, 30), (5, 2, 2, 64, 65), (4, 1, 2, 100, 36), (7, 2, 2, 128, 128),
         (260, 2, 4, 9, 131), (130, 8, 8, 40, 100)]


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32])
@pytest.mark.parametrize('shape', STEPS)
def test_steps_follow_the_sequence(rule, shape, dtype):
    B, Hk, Hv, K, V = shape
    q, k, v, g, beta, s0 = R.delta_inputs(B, 3, Hk, Hv, K, V, dtype, seed=11)
    state = s0.clone()
    os = [rule.gated_delta_step(q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], state) for t in range(3)]
    wo, wf = R.delta_rule(*(x.cpu() for x in (q, k, v, g, beta)), initial=s0.cpu())
    R.assert_close('state', state, wf, R.f32_atol(K + 128))
    R.assert_close('o', torch.stack(os, 1), wo, R.f32_atol(K + 128))


@pytest.mark.parametrize('K', [30, 64, 128])
def test_steps_of_many_states(rule, K):
    """More states than the caches hold, which are passed by; the first and last streams are compared."""
    B, H, V = 64 * 128 // K, 16, 260
    q, k, v, g, beta, s0 = R.delta_inputs(B, 1, H, H, K, V, BF16, seed=31)
    assert B * H * K * V > 32 << 20
    state = s0.clone()
    o = rule.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], state)
    at = [0, 1, B // 2, B - 1]
    wo, wf = R.delta_rule(*(x[at].cpu() for x in (q, k, v, g, beta)), initial=s0[at].cpu())
    R.assert_close('state', state[at], wf, R.f32_atol(K + 128))
    R.assert_close('o', o[at], wo[:, 0], R.f32_atol(K + 128))


@pytest.mark.parametrize('wide', [torch.int32, torch.int64])
def test_step_slots(rule, wide):
    """A pool larger than the batch in any order, idle rows, and refused rows: outside the pool, or named before."""
    B, K, V = 7, 16, 24
    q, k, v, g, beta, _ = R.delta_inputs(B, 1, 1, 2, K, V, BF16, seed=12)
    pool = torch.randn(6, 2, K, V, device='cuda')
    was = pool.clone()
    slots = torch.tensor([4, -1, 0, 6, 4, 5, -9], dtype=wide, device='cuda')
    o = rule.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], pool, slots=slots)
    live = [0, 2, 5]
    at = slots[live].long()
    wo, wf = R.delta_rule(*(x[live].cpu() for x in (q, k, v, g, beta)), initial=was[at].cpu())
    R.assert_close('state', pool[at], wf, R.f32_atol(K + 128))
    R.assert_close('o', o[live], wo[:, 0], R.f32_atol(K + 128))
    assert torch.equal(pool[[1, 2, 3]], was[[1, 2, 3]])
    assert (o[[1, 6]] == 0).all() and torch.isnan(o[[3, 4]]).all()


def test_step_strides(rule):
    B, H, K, V = 3, 2, 24, 20
    q, k, v, g, beta, s0 = R.delta_inputs(B, 2, H, H, K, V, FP32, seed=13)
    store = torch.zeros(H, B, K, V, device='cuda')
    state = store.transpose(0, 1)
    state.copy_(s0)
    o = rule.gated_delta_step(q[:, 1], k[:, 1], v[:, 1], g[:, 1], beta[:, 1], state)
    wo, wf = R.delta_rule(*(x[:, 1:].cpu() for x in (q, k, v, g, beta)), initial=s0.cpu())
    R.assert_close('state', state, wf, R.f32_atol(K + 128))
    R.assert_close('o', o, wo[:, 0], R.f32_atol(K + 128))


# ---------------------------------------------------------------------------------------- streams and captured calls

def test_captured_and_replayed(rule):
    q, k, v, g, beta, s0 = R.delta_inputs(2, 100, 1, 2, 32, 32, BF16, seed=14)
    tok = [x[:, 0].clone() for x in (q, k, v, g, beta)]
    state = s0.clone()
    eager = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    rule.gated_delta_step(*tok, state)
    graph = torch.cuda.CUDAGraph()
    state.copy_(s0)
    with torch.cuda.graph(graph):
        o, final = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
        y = rule.gated_delta_step(*tok, state)
    for i in range(3):
        state.copy_(s0)
        v.mul_(1.0 if i == 0 else -1.0)   # new inputs in the same place
        graph.replay()
        want = rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
        check = s0.clone()
        wy = rule.gated_delta_step(*tok, check)
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(final, want[1])
        assert torch.equal(y, wy) and torch.equal(state, check)
    assert not torch.equal(eager[0], torch.zeros_like(eager[0]))


def test_two_streams_at_once(rule):
    a = R.delta_inputs(1, 500, 2, 2, 64, 64, BF16, seed=15)
    b = R.delta_inputs(1, 500, 2, 2, 64, 64, BF16, seed=16)
    want = [rule.gated_delta_rule(*x[:5], initial_state=x[5]) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(rule.gated_delta_rule(*x[:5], initial_state=x[5]))
    torch.cuda.synchronize()
    for i, (o, final) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(final, want[i % 2][1])
