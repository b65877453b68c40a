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

import numpy as np
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


def assert_close(name, got, want, atol, more=None):
    """|got - want| <= half a step of got's type + atol * rms(want) (+ more), element by element; NaN and inf in the same
    places."""
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
    if more is not None:   # half a step of a value that is off by `more` itself
        bound = bound + more.double().cpu()[fin] * (1 + torch.finfo(got.dtype).eps / 2)
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


def philox_bits(n, seed, offset):
    """16 random bits for each of n elements as blocks/dropout.py defines them: Philox4x32-10 in unsigned 64-bit numpy."""
    u, low, half = np.uint64, np.uint64(0xffffffff), np.uint64(32)
    c = np.arange(-(-n // 8), dtype=u)
    x = [c & low, c >> half, np.full_like(c, offset & 0xffffffff), np.full_like(c, (offset >> 32) & 0xffffffff)]
    k = [seed & 0xffffffff, (seed >> 32) & 0xffffffff]
    for _ in range(10):
        a, b = x[0] * u(0xD2511F53), x[2] * u(0xCD9E8D57)
        x = [(b >> half) ^ x[1] ^ u(k[0]), b & low, (a >> half) ^ x[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return np.stack([v >> s & u(0xffff) for v in x for s in (u(0), u(16))], 1).reshape(-1)[:n]


def dropout(x, p, seed, offset=0, residual=None):
    below = int(round(p * 65536))
    keep = torch.from_numpy(philox_bits(x.numel(), seed, offset).astype(np.int64) >= below).reshape(x.shape)
    y = torch.where(keep, x.double().cpu() * (65536 / max(65536 - below, 1)), 0.0)
    return (y if residual is None else y + residual.double().cpu()), keep


def gated_unit(x, wg, wu, activation):
    x, wg, wu = x.double(), wg.double(), wu.double()
    a, b = x @ wg, x @ wu
    f = {'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu, 'sigmoid': torch.sigmoid}[activation]
    return f(a) * b


def unit_atol(n):
    """y: two f32 sums of n products, an activation with slope at most 1.13 and size at most |a|, and their product, whose size the
    two sums' root mean squares bound: three times the bound of one sum."""
    return 3 * f32_atol(n)


def unit_grad_bounds(x, wg, wu, dy, activation):
    """What dx, dwg and dwu may be off by, element by element, beyond their own rounding.  They are sums of products whose operands
    da and db were rounded to the type, half a step h relative each: at most h times the sum of the terms' sizes, which is formed here
    (|da| |Wg|^T + |db| |Wu|^T, |x|^T |da|, |x|^T |db|).  The f32 sums of n terms add n 2^-24 of the same, and the projections' errors
    (f32 sums over D) 2^-24 (n + D) of the gradients' root mean square, three times (as for y)."""
    half = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 0.0
    x, wg, wu, dy = (t.detach().double().cpu() for t in (x, wg, wu, dy))
    a, b = (x @ wg).requires_grad_(), (x @ wu).requires_grad_()
    f = {'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu, 'sigmoid': torch.sigmoid}[activation]
    da, db = (t.abs() for t in torch.autograd.grad(f(a) * b, (a, b), dy))
    sizes = (da @ wg.abs().t() + db @ wu.abs().t(), x.abs().t() @ da, x.abs().t() @ db)
    terms = (2 * wg.size(1), x.size(0), x.size(0))
    return [((half + n * 2.0 ** -24) * s, 3 * f32_atol(n + x.size(1))) for s, n in zip(sizes, terms)]
