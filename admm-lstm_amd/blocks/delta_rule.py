"""The gated delta rule: a gated recurrence with a matrix state, beside the LSTM cell of ``blocks/lstm.py``.

For each sequence and value head, with the state S [K, V] (float32)::

    S' = exp(g_t) S;   u_t = beta_t (v_t - S'^T k_t);   S = S' + k_t u_t^T;   o_t = scale S^T q_t

``gated_delta_rule`` runs whole sequences (training and prompts) and carries gradients; ``gated_delta_step`` runs one
token of each of many streams and updates their states in place (serving).  Both need HIP device tensors and run in
libseqops.so (hand-written gfx950 kernels) on the current stream of the tensors' device.

All of it can be captured into a graph.  As with PyTorch's own operators, a backward pass is captured only while no eager
autograd graph of the same leaves is alive (it would tie the captured work to the stream of the eager one).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from admm_amd import _seq_native

_E = _seq_native.entry_points()


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                     scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                     offsets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Outputs o [B, T, Hv, V] and final states [B, Hv, K, V] (float32) of whole sequences.

    q, k [B, T, Hk, K] and v [B, T, Hv, V] of one type (bfloat16, float16, float32), K <= 128, Hv a multiple of Hk (value
    head h uses query/key head h // (Hv // Hk)); g [B, T, Hv] (the log of the decay) and beta [B, T, Hv] float32.  Any
    strides.  ``scale`` defaults to K ** -0.5, ``initial_state`` [B, Hv, K, V] float32 to zeros.

    ``offsets`` (int32 or int64 on the device, non-decreasing, within [0, T]) packs sequences of different lengths into
    B = 1: sequence n is rows ``offsets[n]:offsets[n + 1]``, and states are [len(offsets) - 1, Hv, K, V].  A sequence may
    be empty; rows outside every sequence get zeros.

    Sums and states are float32, and products accurate to float32 (operands split into three bf16 pieces), but for what only
    results of 16 bits are made of: o of such inputs takes 16 bits (two pieces) of the state and of the rows written, and dq and dk
    16 bits of the rows' weights.  o and the gradients of q, k, v are rounded to the inputs' type.  A row whose g is -inf starts its
    sequence's state afresh.  Where rows grow (g > 0), exp of their sum over 64 rows has to be within float32.  Any other value that
    is not finite (or is above 3.39e38) makes NaN what depends on it, and nothing before its row (in q: o of that row; in v: its
    column from that row on; in k, g and beta: all columns from that row on).
    """
    return _E.gated_delta_rule(q, k, v, g, beta, scale, initial_state, offsets)


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, *, scale: Optional[float] = None,
                     slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each of B streams: returns o [B, Hv, V] and replaces the streams' states in place.

    q, k [B, Hk, K], v [B, Hv, V], g, beta [B, Hv] as in ``gated_delta_rule``; ``state`` float32 [B, Hv, K, V], or a pool
    [P, Hv, K, V] of which row b uses ``state[slots[b]]`` (int32 or int64 on the device).  A negative slot marks an idle row
    (a batch padded for a captured graph): its output is zero and no state changes.  A slot outside the pool, or one that an
    earlier row of the batch names too, gives NaN in that row's output and changes no state.  Carries no gradients.
    """
    return _E.gated_delta_step(q, k, v, g, beta, state, scale, slots)
