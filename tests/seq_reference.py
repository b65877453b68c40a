"""Plain 64-bit implementations of the sequence-layer operators and the tolerances that their tests use.

Tolerances, from the arithmetic:

* a value rounded to type t is off by at most half a step, finfo(t).eps / 2 relative to the value;
* an f32 sum of n products is off by at most about n 2^-24 of the sum of the terms' sizes (each of the n additions and the
  operands' three-plane split, 2^-24 each); the terms' sizes add up to at most sqrt(n) times the root mean square of such sums
  (Cauchy-Schwarz, rows of independent signs).  With n = K + 128 inner values (two 64-row products and one of length K) the
  part that does not shrink with the value is F32_TERMS(n) = 2^-24 n of the tensor's root mean square, doubled for the passage
  through the chunk's triangular system, whose inverse has norm below 2 for the tests' inputs;
* what only a 16-bit o is made of keeps two bf16 planes of S, u and P (2^-17 each, so 3 * 2^-17 of the terms' sizes, which are at
  most sqrt(K + 64) times the root mean square).
"""
import math

import torch


def f32_atol(n):
    return 2.0 * n * 2.0 ** -24


def o_atol(dtype, K):
    if dtype == torch.float32:
        return f32_atol(K + 128)
    return 3 * 2.0 ** -17 * math.sqrt(K + 64) + f32_atol(K + 128)


def grad_atol(dtype, K, V):
    """Gradients: sums over K, V and the chunk's 64 rows several times over.  dbeta and dg add up to six such sums that partly
    cancel, each of up to the size of the tensor's larger values: four times the bound of one."""
    atol = 4 * f32_atol(K + V + 256)
    return atol if dtype == torch.float32 else atol + 3 * 2.0 ** -17 * math.sqrt(K + 64)


def assert_close(name, got, want, atol):
    """|got - want| <= half a step of got's type + atol * rms(want), element by element; NaN and inf in the same places."""
    assert got.shape == want.shape, f'{name}: shape {tuple(got.shape)} != {tuple(want.shape)}'
    g, w = got.double().cpu(), want.double().cpu()
    assert torch.equal(torch.isfinite(g), torch.isfinite(w)), f'{name}: non-finite values in other places'
    fin = torch.isfinite(w)
    assert torch.equal(g[~fin].nan_to_num(7.0), w[~fin].nan_to_num(7.0)), f'{name}: non-finite values differ'
    g, w = g[fin], w[fin]
    if not g.numel():
        return
    rms = float(w.square().mean().sqrt())
    bound = torch.finfo(got.dtype).eps / 2 * w.abs() + atol * rms
    over = ((g - w).abs() - bound).max()
    assert float(over) <= 0, (f'{name}: off by up to {float((g - w).abs().max()):.3e} (rms {rms:.3e}), '
                              f'{float(over):.3e} more than allowed')


def delta_rule(q, k, v, g, beta, scale=None, initial=None, offsets=None):
    """Token by token in float64, differentiable.  Arguments as blocks.delta_rule.gated_delta_rule (any device)."""
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    B, T, Hk, K = q.shape
    Hv, V = v.shape[2:]
    scale = K ** -0.5 if scale is None else scale
    q, k = (x.repeat_interleave(Hv // Hk, 2) for x in (q, k))
    if offsets is None:
        spans = [(b, 0, T) for b in range(B)]
    else:
        off = offsets.tolist()
        spans = [(0, a, e) for a, e in zip(off, off[1:])]
    o, finals = torch.zeros(B, T, Hv, V, dtype=torch.float64, device=q.device), []
    pieces = []
    for i, (b, a, e) in enumerate(spans):
        S = (torch.zeros(Hv, K, V, dtype=torch.float64, device=q.device) if initial is None else initial[i].double())
        rows = []
        for t in range(a, e):
            S = S * g[b, t].exp()[:, None, None]
            u = beta[b, t][:, None] * (v[b, t] - (S * k[b, t][:, :, None]).sum(1))
            S = S + k[b, t][:, :, None] * u[:, None, :]
            rows.append(scale * (S * q[b, t][:, :, None]).sum(1))
        finals.append(S)
        if rows:
            pieces.append((b, a, e, torch.stack(rows)))
    for b, a, e, r in pieces:
        o = o.index_put((torch.tensor(b), torch.arange(a, e)), r)
    final = torch.stack(finals) if finals else torch.zeros(0, Hv, K, V, dtype=torch.float64, device=q.device)
    return o, final


def delta_inputs(B, T, Hk, Hv, K, V, dtype, seed=0, n=None, device='cuda'):
    """q, k of length one, v, decays between 1e-3 and 1, write strengths in (0, 1), initial states."""
    gen = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen)

    def unit(x):
        return x / x.norm(dim=-1, keepdim=True).clamp_min(1e-3)

    q, k, v = unit(randn(B, T, Hk, K)), unit(randn(B, T, Hk, K)), randn(B, T, Hv, V)
    g = -torch.exp(math.log(1e-3) * torch.rand(B, T, Hv, generator=gen))
    beta = torch.sigmoid(randn(B, T, Hv))
    s0 = 0.5 * randn(B if n is None else n, Hv, K, V)
    return [x.to(device) for x in (q.to(dtype), k.to(dtype), v.to(dtype), g, beta, s0)]
