"""The sequence operators as a network uses them: a residual layer of the delta rule and the gated unit, with dropout, in training
and token by token; and the LSTM that drops part of its last state."""
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu

B, T, D, HK, HV, K, V, F = 2, 70, 48, 2, 4, 16, 24, 80
P, SEED = 0.1, 1234

# One f32 result of the layer passes through sums of at most T (K + V) + 3 D + F products one inside the other; each rounding is
# 2^-24 of a partial sum, and partial sums are of the results' size (weights are scaled to keep the root mean square).  The bound
# adds all roundings up, which is far above what they come to at random.
ATOL = (T * (K + V) + 3 * D + F) * 2.0 ** -24


def _weights():
    gen = torch.Generator().manual_seed(7)

    def w(a, b):
        return (torch.randn(a, b, generator=gen) / a ** 0.5).cuda()

    return dict(q=w(D, HK * K), k=w(D, HK * K), v=w(D, HV * V), g=w(D, HV), b=w(D, HV), o=w(HV * V, D), gate=w(D, F), up=w(D, F), down=w(F, D))


def _project(x, w):
    """q, k of length one, v, g < 0, beta, from x [..., D]."""
    q, k = ((x @ w[n]).unflatten(-1, (HK, K)) for n in 'qk')
    q, k = (t / t.norm(dim=-1, keepdim=True) for t in (q, k))
    g, beta = -torch.nn.functional.softplus(x @ w['g']), torch.sigmoid(x @ w['b'])
    return q, k, (x @ w['v']).unflatten(-1, (HV, V)), g, beta


def _layer(x, w, s0, rule, unit, drop):
    o, s1 = rule(*_project(x, w), s0)
    y = drop(o.flatten(-2) @ w['o'], 0, x)
    return drop(unit(y, w['gate'], w['up']) @ w['down'], 1, y), s1


def _own(x, w, s0, p=P):
    from blocks import delta_rule, dropout, gated_unit
    return _layer(x, w, s0, lambda q, k, v, g, b, s: delta_rule.gated_delta_rule(q, k, v, g, b, initial_state=s),
                  gated_unit.gated_unit, lambda t, offset, res: dropout.dropout(t, p, SEED, offset=offset, residual=res))


def _plain(x, w, s0, p=P):
    def drop(t, offset, res):
        keep = R.dropout(t.detach(), p, SEED, offset)[1]
        return torch.where(keep, t / (1 - round(p * 65536) / 65536), torch.zeros_like(t)) + res

    return _layer(x, w, s0, lambda q, k, v, g, b, s: R.delta_rule(q, k, v, g, b, initial=s),
                  lambda t, a, b: R.gated_unit(t, a, b, 'silu'), drop)


def _inputs(T):
    gen = torch.Generator().manual_seed(8)
    return torch.randn(B, T, D, generator=gen).cuda(), (0.5 * torch.randn(B, HV, K, V, generator=gen)).cuda()


@pytest.mark.parametrize('T', [70, 20])
def test_a_layer_in_training(T):
    x, s0 = _inputs(T)
    w = _weights()
    leaves = [t.requires_grad_() for t in (x, s0, *w.values())]
    y, s1 = _own(x, w, s0)
    dy, ds = torch.randn_like(y), torch.randn_like(s1)
    got = torch.autograd.grad([y, s1], leaves, [dy, ds])
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    wy, ws = _plain(ref[0], dict(zip(w, ref[2:])), ref[1])
    want = torch.autograd.grad([wy, ws], ref, [dy.cpu().double(), ds.cpu().double()])
    R.assert_close('y', y.detach(), wy.detach(), ATOL)
    R.assert_close('state', s1.detach(), ws.detach(), ATOL)
    for n, a, b in zip(('x', 's0', *w), got, want):
        R.assert_close('d' + n, a, b, 4 * ATOL)   # forward once, and as long a way back, for each of two uses of a value


def test_token_by_token_follows_the_sequence():
    """A prompt in one call, then single tokens from its state, against the whole sequence in one call."""
    from blocks import delta_rule, gated_unit
    x, s0 = _inputs(T)
    w = _weights()
    with torch.no_grad():
        whole, final = _own(x, w, s0, p=0.0)
        head, state = _own(x[:, :60], w, s0, p=0.0)
        R.assert_close('prompt', head, whole[:, :60].cpu(), ATOL)
        for t in range(60, T):
            y = x[:, t] + delta_rule.gated_delta_step(*_project(x[:, t], w), state).flatten(-2) @ w['o']
            y = y + gated_unit.gated_unit(y, w['gate'], w['up']) @ w['down']
            R.assert_close(f'token {t}', y, whole[:, t].cpu(), 2 * ATOL)
        R.assert_close('state', state, final.cpu(), 2 * ATOL)


def test_captured_training_of_a_layer():
    """The layer's forward and backward in one graph, the dropout's seed read from the device at each replay."""
    from blocks import delta_rule, dropout, gated_unit
    x, s0 = _inputs(T)
    w = _weights()
    seed = torch.tensor(5, dtype=torch.int64, device='cuda')
    leaves = [t.requires_grad_() for t in (x, s0, *w.values())]

    def step():
        y, s1 = _layer(x, w, s0, lambda q, k, v, g, b, s: delta_rule.gated_delta_rule(q, k, v, g, b, initial_state=s),
                       gated_unit.gated_unit, lambda t, offset, res: dropout.dropout(t, P, seed, offset=offset, residual=res))
        return (y, s1, *torch.autograd.grad([y, s1], leaves, [torch.ones_like(y), torch.ones_like(s1)]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        seed.add_(1)
        graph.replay()
        y = out[0].clone()
        want = step()[0]
        torch.cuda.synchronize()
        assert torch.equal(y, want), i   # (the weights' gradients pass through library products, whose sums may differ in order)


def test_lstm_drops_part_of_its_last_state():
    from blocks.dropout import dropout
    from blocks.lstm import LSTM
    torch.manual_seed(3)
    m = LSTM(5, 32, 4, with_grad=True, dropout=0.25).cuda()
    torch.manual_seed(3)
    plain = LSTM(5, 32, 4, with_grad=True).cuda()
    assert all(torch.equal(a, b) for a, b in zip(m.parameters(), plain.parameters()))
    x = torch.randn(9, 6, 5, device='cuda')
    m.eval()
    assert torch.equal(m(x), plain(x))
    m.train()
    seed = torch.tensor(77, device='cuda')
    y = m(x, dropout_seed=seed)
    keep = R.dropout(torch.zeros(9, 32), 0.25, 77)[1].cuda()
    with torch.no_grad():
        eye = LSTM(5, 32, 32, with_grad=True).cuda()
        for n, p in plain.named_parameters():
            if n != 'out':
                eye.get_parameter(n).copy_(p)
        eye.out.copy_(torch.eye(32))
        h = eye(x)   # the last state itself: a product with ones and zeros is exact
        assert torch.equal(y, dropout(h, 0.25, seed) @ m.out) and torch.equal(dropout(h, 0.25, seed) != 0, keep & (h != 0))
    y.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    torch.manual_seed(11)
    a, b = m(x), m(x)
    torch.manual_seed(11)
    assert torch.equal(m(x), a) and not torch.equal(a, b)   # a new mask each call, from torch's generator


def test_what_the_gradients_need_is_freed_with_them():
    """The work memory and the kept projections go after the backward pass, though the results (and their graph) live on."""
    from blocks import delta_rule, gated_unit
    q, k, v, g, beta, s0 = R.delta_inputs(2, 2048, 4, 4, 64, 64, torch.bfloat16, seed=70)
    v.requires_grad_()
    x, w = torch.randn(4096, 64, device='cuda', requires_grad=True), torch.randn(64, 512, device='cuda')
    for call, leaf in ((lambda: delta_rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)[0], v), (lambda: gated_unit.gated_unit(x, w, w), x)):
        torch.autograd.grad(call().sum(), leaf)
        before = torch.cuda.memory_allocated()
        y = call()
        held = torch.cuda.memory_allocated() - before
        torch.autograd.grad(y.sum(), leaf)
        after = torch.cuda.memory_allocated() - before
        assert after <= held / 2 and after <= 2 * y.numel() * y.element_size()   # y itself (and its final state)


def test_inference_mode():
    """Results as under no_grad; a state made there is refused outside, before it is written."""
    from blocks import delta_rule
    q, k, v, g, beta, s0 = R.delta_inputs(2, 40, 1, 2, 16, 16, torch.float32, seed=71)
    with torch.no_grad():
        want = delta_rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
    with torch.inference_mode():
        o, state = delta_rule.gated_delta_rule(q, k, v, g, beta, initial_state=s0)
        assert torch.equal(o, want[0]) and torch.equal(state, want[1])
        kept = state.clone()
        first = delta_rule.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], state)
    assert torch.isfinite(first).all() and not torch.equal(state, kept)
    kept = state.clone()
    with pytest.raises(RuntimeError, match='nference'):
        delta_rule.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0], state)
    assert torch.equal(state, kept)


def test_rows_expanded_from_one():
    """Rows and gradients whose stride is zero."""
    from blocks import gated_unit
    row, w, u = torch.randn(1, 64, device='cuda'), torch.randn(64, 72, device='cuda'), torch.randn(64, 72, device='cuda')
    for M in (7, 100):
        x = row.expand(M, 64).requires_grad_()
        y = gated_unit.gated_unit(x, w, u)
        assert torch.equal(y, y[:1].expand(M, 72))
        one = torch.randn(1, 72, device='cuda')
        (a,) = torch.autograd.grad(y, x, one.expand(M, 72), retain_graph=True)
        (b,) = torch.autograd.grad(y, x, one.expand(M, 72).contiguous())
        assert torch.equal(a, b)


def test_two_threads_at_once():
    """Calls from two threads on streams of their own."""
    import threading
    from blocks import delta_rule
    ins = [R.delta_inputs(2, T, 1, 2, 32, 32, torch.bfloat16, seed=72 + T) for T in (30, 200)]
    want = [delta_rule.gated_delta_rule(*i[:5], initial_state=i[5]) for i in ins]
    torch.cuda.synchronize()
    got = [None, None]

    def work(n):
        with torch.cuda.stream(torch.cuda.Stream()), torch.no_grad():
            for _ in range(20):
                got[n] = delta_rule.gated_delta_rule(*ins[n][:5], initial_state=ins[n][5])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
