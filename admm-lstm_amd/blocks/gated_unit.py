"""The gated unit ``y = act(x Wg) * (x Wu)``: the wide layer between recurrent layers.

One fused kernel forms both projections, the activation and the product; the gradients are tiled matrix products as well.
Weights are [D, F] like the LSTM's ``x2q`` (``blocks/lstm.py``), whose product i * g is such a unit.  Runs in libseqops.so
(hand-written gfx950 kernels) on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from admm_amd import _seq_native as N

ACTIVATIONS = {'silu': 0, 'gelu': 1, 'sigmoid': 2}
MAX = 1 << 20


def _row_stride(t):
    return t.stride(0) if t.size(0) > 1 else t.size(1)


class _Call:
    """The C descriptor of one call and the tensors it points into (x as [M, D])."""

    def __init__(self, x, wg, wu, act):
        self.x, self.wg, self.wu = x, wg, wu = N.rows_last(x), N.rows_last(wg), N.rows_last(wu)
        self.u = N.SeqUnit(x.size(0), x.size(1), wg.size(1), act, N.DTYPES[x.dtype], x.device.index, x.data_ptr(),
                           wg.data_ptr(), wu.data_ptr(), _row_stride(x), _row_stride(wg), _row_stride(wu))

    def work(self, backward):
        need = ctypes.c_int64()
        N.check(N.load().seq_unit_workspace(ctypes.byref(self.u), backward, ctypes.byref(need)), 'gated_unit')
        return torch.empty(need.value, dtype=torch.uint8, device=self.x.device)

    def forward(self, keep):
        M, F, dev = self.x.size(0), self.wg.size(1), self.x.device
        y = torch.empty(M, F, dtype=self.x.dtype, device=dev)
        pre = torch.empty(2, M, F, dtype=torch.float32, device=dev) if keep else None
        work = self.work(False)
        N.check(N.load().seq_unit_forward(ctypes.byref(self.u), work.data_ptr(), work.numel(), y.data_ptr(),
                                          pre.data_ptr() if keep else None, N.stream(dev)), 'gated_unit')
        return y, pre


class _GatedUnit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, act):
        y, ctx.pre = _Call(x, wg, wu, act).forward(True)
        ctx.save_for_backward(x, wg, wu)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, wg, wu = ctx.saved_tensors
        call, dev, dy = _Call(x, wg, wu, ctx.act), x.device, N.rows_last(dy)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = (torch.empty(2, *wg.shape, dtype=wg.dtype, device=dev)
              if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else (None, None))
        work = call.work(True)
        N.check(N.load().seq_unit_backward(ctypes.byref(call.u), work.data_ptr(), work.numel(), ctx.pre.data_ptr(),
                                           dy.data_ptr(), _row_stride(dy),
                                           *(t.data_ptr() if t is not None else None for t in (dx, dw[0], dw[1])),
                                           N.stream(dev)), 'gated_unit backward')
        return dx, dw[0], dw[1], None


def gated_unit(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str = 'silu') -> torch.Tensor:
    """``act(x @ w_gate) * (x @ w_up)`` for x [..., D] and weights [D, F], all of one type (bfloat16, float16, float32).

    ``activation``: 'silu', 'gelu' (the exact one) or 'sigmoid'.  Any strides.  Products are summed in float32 (float32
    operands are split into bf16 pieces, accurate to float32) and rounded once; gradients reach x and both weights, and keep the
    two projections in float32 (8 bytes for each of M x F values) from the forward pass.
    """
    N.require_tensors(x=x, w_gate=w_gate, w_up=w_up)
    N.require(x.dtype in N.DTYPES, f'x must be bfloat16, float16 or float32 (got {x.dtype})')
    N.require(activation in ACTIVATIONS, f'activation must be one of {", ".join(ACTIVATIONS)} (got {activation!r})')
    N.require(x.dim() >= 1, 'x must have at least one axis')
    for name, w in (('w_gate', w_gate), ('w_up', w_up)):
        N.require(w.dtype == x.dtype, f'{name} must have the type of x, {x.dtype} (got {w.dtype})')
        N.require(w.dim() == 2 and w.size(0) == x.size(-1), f'{name} must be [{x.size(-1)}, F] (got {tuple(w.shape)})')
    N.require(w_gate.shape == w_up.shape, f'w_gate and w_up differ in shape: {tuple(w_gate.shape)}, {tuple(w_up.shape)}')
    D, F = w_gate.shape
    N.require(1 <= D <= MAX and 1 <= F <= MAX, f'weights must be between 1 x 1 and {MAX} x {MAX} (got {D} x {F})')
    N.require_device(x=x, w_gate=w_gate, w_up=w_up)
    act = ACTIVATIONS[activation]
    rows = x.reshape(-1, D)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        y = _GatedUnit.apply(rows, w_gate, w_up, act)
    else:
        y = _Call(rows, w_gate, w_up, act).forward(False)[0]
    return y.view(*x.shape[:-1], F)
