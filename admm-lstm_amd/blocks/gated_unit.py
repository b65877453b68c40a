"""The gated unit ``y = act(x Wg) * (x Wu)``: the wide layer between recurrent layers.

One fused kernel forms both projections, the activation and the product; the gradients are tiled matrix products as well.
Weights are [D, F] like the LSTM's ``x2q`` (``blocks/lstm.py``), whose product i * g is such a unit.  Runs in libseqops.so
(hand-written gfx950 kernels) on the current stream of the tensors' device.
"""
from __future__ import annotations

import torch

from admm_amd import _seq_native

_E = _seq_native.entry_points()


def gated_unit(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str = 'silu') -> torch.Tensor:
    """``act(x @ w_gate) * (x @ w_up)`` for x [..., D] and weights [D, F], all of one type (bfloat16, float16, float32).

    ``activation``: 'silu', 'gelu' (the exact one) or 'sigmoid'.  Any strides.  Products are summed in float32 and rounded once
    (float32 operands are split into bf16 pieces, accurate to float32; an infinite operand counts as NaN there, and in the gradients
    of float16).  Gradients reach x and both weights, and keep the two projections in float32 (8 bytes for each of M x F values)
    from the forward pass.  They are products of the projections' gradients, which bfloat16 holds in bfloat16 (a second rounding)
    and float16 in 16 bits with the range of float32 (three products where bfloat16 takes one).
    """
    return _E.gated_unit(x, w_gate, w_up, activation)
