"""A captured training step of a whole layer of the sequence operators: every result of every replay."""
import pytest
import torch

import seq_reference as R
from test_gpu_seq_together import ATOL, P, T, _inputs, _layer, _weights

pytestmark = pytest.mark.gpu


def test_all_results_of_a_captured_layer():
    """The final state is the operator's own and equal; the gradients pass through library products, whose sums may differ in order (as
    far as one of two results of the layer may be from the true one, twice)."""
    from blocks import delta_rule, dropout, gated_unit
    x, s0 = _inputs(T)
    w = _weights()
    seed = torch.tensor(5, dtype=torch.int64, device='cuda')
    leaves = [t.requires_grad_() for t in (x, s0, *w.values())]

    def step():
        y, s1 = _layer(x, w, s0, lambda q, k, v, g, b, s: delta_rule.gated_delta_rule(q, k, v, g, b, initial_state=s),
                       gated_unit.gated_unit, lambda t, offset, res: dropout.dropout(t, P, seed, offset=offset, residual=res))
        return [t.detach() for t in (y, s1, *torch.autograd.grad([y, s1], leaves, [torch.ones_like(y), torch.ones_like(s1)]))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    last = None
    for i in range(3):
        seed.add_(1)
        with torch.no_grad():
            s0.mul_(-0.5)
        graph.replay()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        for n, a, b in zip(('x', 's0', *w), got[2:], want[2:]):
            R.assert_close(f'd{n}, replay {i}', a, b.cpu(), 2 * 4 * ATOL)
        if last:   # other masks: other results, but for the final state, which has none in it (and has forgotten its start)
            assert not [n for n, a, b in zip(('y', 's1', 'x', 's0', *w), got, last) if n != 's1' and torch.equal(a, b)], i
        last = got
