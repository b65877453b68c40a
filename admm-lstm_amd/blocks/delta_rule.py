"""The gated delta rule: a gated recurrence with a matrix state, beside the LSTM cell of ``blocks/lstm.py``.

For each sequence and value head, with the state S [K, V] (float32)::

    S' = exp(g_t) S;   u_t = beta_t (v_t - S'^T k_t);   S = S' + k_t u_t^T;   o_t = scale S^T q_t

``gated_delta_rule`` runs whole sequences (training and prompts) and carries gradients; ``gated_delta_step`` runs one
token of each of many streams and updates their states in place (serving).  Both need HIP device tensors and run in
libseqops.so (hand-written gfx950 kernels) on the current stream of the tensors' device.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from admm_amd import _seq_native as N

MAX_K = 128


def _check_rows(q, k, v, g, beta, lead: int, lead_name: str) -> None:
    N.require(q.dtype in N.DTYPES, f'q must be bfloat16, float16 or float32 (got {q.dtype})')
    for name, t in (('k', k), ('v', v)):
        N.require(t.dtype == q.dtype, f'{name} must have the type of q, {q.dtype} (got {t.dtype})')
    for name, t in (('g', g), ('beta', beta)):
        N.require(t.dtype == torch.float32, f'{name} must be float32 (got {t.dtype})')
    for name, t in (('q', q), ('k', k), ('v', v)):
        N.require(t.dim() == lead + 2, f'{name} must be {lead_name} x heads x values (got shape {tuple(t.shape)})')
    N.require(q.shape == k.shape, f'q and k differ in shape: {tuple(q.shape)} and {tuple(k.shape)}')
    N.require(v.shape[:lead] == q.shape[:lead], f'v has {lead_name} {tuple(v.shape[:lead])}, q {tuple(q.shape[:lead])}')
    for name, t in (('g', g), ('beta', beta)):
        N.require(t.shape == v.shape[:-1], f'{name} must have shape {tuple(v.shape[:-1])} (got {tuple(t.shape)})')
    Hk, Hv = q.size(-2), v.size(-2)
    N.require(Hk > 0 and Hv > 0 and Hv % Hk == 0,
              f'the number of value heads ({Hv}) must be a multiple of that of query/key heads ({Hk})')
    N.require(1 <= q.size(-1) <= MAX_K, f'query/key rows must have 1 to {MAX_K} values (got {q.size(-1)})')
    N.require(v.size(-1) >= 1, 'value rows must not be empty')


def _apart(state: torch.Tensor) -> bool:
    """Whether the [K, V] states of a pool [P, Hv, K, V] are apart in memory."""
    size = state.size(2) * state.size(3)
    for stride, n in sorted((state.stride(i), state.size(i)) for i in (0, 1) if state.size(i) > 1):
        if stride < size:
            return False
        size = stride * n
    return True


class _Call:
    """The C descriptor of one call and the tensors it points into."""

    def __init__(self, q, k, v, g, beta, initial, offsets, scale):
        self.tensors = q, k, v, g, beta, initial, offsets = (
            N.rows_last(q), N.rows_last(k), N.rows_last(v), g, beta, initial, offsets)
        d = self.d = N.SeqDelta()
        d.batch, d.T = q.shape[:2]
        d.sequences = q.size(0) if offsets is None else offsets.numel() - 1
        d.Hk, d.K, d.Hv, d.V = *q.shape[2:], *v.shape[2:]
        d.dtype, d.scale, d.device = N.DTYPES[q.dtype], scale, q.device.index
        d.q, d.k, d.v, d.g, d.beta = (t.data_ptr() for t in (q, k, v, g, beta))
        for name, t in (('q', q), ('k', k), ('v', v), ('g', g), ('beta', beta)):
            getattr(d, name + '_stride')[:] = t.stride()[:3]
        if offsets is not None:
            d.offsets, d.offsets_64 = offsets.data_ptr(), int(offsets.dtype == torch.int64)
        if initial is not None:
            d.initial = initial.data_ptr()

    def forward(self, saved: bool):
        q, v = self.tensors[0], self.tensors[2]
        lib, need = N.load(), ctypes.c_int64()
        N.check(lib.seq_delta_workspace(ctypes.byref(self.d), saved, ctypes.byref(need)), 'gated_delta_rule')
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        o = torch.empty(v.shape, dtype=v.dtype, device=q.device)
        final = torch.empty(self.d.sequences, self.d.Hv, self.d.K, self.d.V, dtype=torch.float32, device=q.device)
        N.check(lib.seq_delta_forward(ctypes.byref(self.d), saved, work.data_ptr(), need.value, o.data_ptr(),
                                      final.data_ptr(), N.stream(q.device)), 'gated_delta_rule')
        return o, final, work


class _GatedDeltaRule(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial, offsets, scale):
        call = _Call(q, k, v, g, beta, initial, offsets, scale)
        o, final, work = call.forward(True)
        ctx.save_for_backward(q, k, v, g, beta, initial, offsets)
        ctx.work, ctx.scale = work, scale
        return o, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, d_final):
        q, k, v, g, beta, initial, offsets = ctx.saved_tensors
        call = _Call(q, k, v, g, beta, initial, offsets, ctx.scale)
        lib, need, dev = N.load(), ctypes.c_int64(), q.device
        N.check(lib.seq_delta_backward_scratch(ctypes.byref(call.d), ctypes.byref(need)), 'gated_delta_rule')
        scratch = torch.empty(need.value, dtype=torch.uint8, device=dev)
        d_o, d_final = d_o.contiguous(), d_final.contiguous()
        dq, dk, dv, dg, dbeta = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v, g, beta))
        d_initial = torch.empty_like(d_final) if ctx.needs_input_grad[5] else None
        N.check(lib.seq_delta_backward(ctypes.byref(call.d), ctx.work.data_ptr(), ctx.work.numel(), scratch.data_ptr(),
                                       need.value, d_o.data_ptr(), d_final.data_ptr(),
                                       *(t.data_ptr() for t in (dq, dk, dv, dg, dbeta)),
                                       d_initial.data_ptr() if d_initial is not None else None, N.stream(dev)),
                'gated_delta_rule backward')
        return dq, dk, dv, dg, dbeta, d_initial, None, None


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

    Products and states are float32 throughout (operands split into bf16 pieces); only o and gradients of q, k, v are
    rounded to the inputs' type.  A row whose g is -inf starts its sequence's state afresh.  Any other value that is not
    finite makes NaN what depends on it, and nothing before its row (in q: o of that row; in v: its column from that row on;
    in k, g and beta: all columns from that row on).
    """
    N.require_tensors(q=q, k=k, v=v, g=g, beta=beta, initial_state=initial_state, offsets=offsets)
    _check_rows(q, k, v, g, beta, 2, 'batch x time')
    n = q.size(0)
    if offsets is not None:
        N.require(q.size(0) == 1, f'packed sequences need a batch of 1 (got {q.size(0)})')
        N.require(offsets.dim() == 1 and offsets.numel() >= 1 and offsets.dtype in (torch.int32, torch.int64),
                  f'offsets must be a vector of int32 or int64 (got {offsets.dtype}, shape {tuple(offsets.shape)})')
        offsets, n = offsets.contiguous(), offsets.numel() - 1
    if initial_state is not None:
        want = (n, v.size(2), q.size(3), v.size(3))
        N.require(initial_state.dtype == torch.float32 and tuple(initial_state.shape) == want,
                  f'initial_state must be float32 of shape {want} (got {initial_state.dtype}, '
                  f'{tuple(initial_state.shape)})')
        initial_state = initial_state.contiguous()
    N.require_device(q=q, k=k, v=v, g=g, beta=beta, initial_state=initial_state, offsets=offsets)
    scale = q.size(3) ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state)):
        return _GatedDeltaRule.apply(q, k, v, g, beta, initial_state, offsets, scale)
    return _Call(q, k, v, g, beta, initial_state, offsets, scale).forward(False)[:2]


@torch.no_grad()
def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, *, scale: Optional[float] = None,
                     slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each of B streams: returns o [B, Hv, V] and replaces the streams' states in place.

    q, k [B, Hk, K], v [B, Hv, V], g, beta [B, Hv] as in ``gated_delta_rule``; ``state`` float32 [B, Hv, K, V], or a pool
    [P, Hv, K, V] of which row b uses ``state[slots[b]]`` (int32 or int64 on the device).  A negative slot marks an idle row
    (a batch padded for a captured graph): its output is zero and no state changes.  A slot outside the pool, or one that an
    earlier row of the batch names too, gives NaN in that row's output and changes no state.  Carries no gradients.
    """
    N.require_tensors(q=q, k=k, v=v, g=g, beta=beta, state=state, slots=slots)
    _check_rows(q, k, v, g, beta, 1, 'batch')
    B, Hk, K = q.shape
    Hv, V = v.shape[1:]
    N.require(state.dtype == torch.float32 and state.dim() == 4 and tuple(state.shape[1:]) == (Hv, K, V),
              f'state must be float32 of shape (states, {Hv}, {K}, {V}) (got {state.dtype}, {tuple(state.shape)})')
    N.require(state.stride(3) == 1 and state.stride(2) == V or state.numel() == 0,
              'the last two axes of state must be contiguous (it is updated in place)')
    N.require(_apart(state), 'the states overlap in memory (an expanded tensor?): they are updated in place')
    if slots is None:
        N.require(state.size(0) == B, f'{B} rows need {B} states (got {state.size(0)}); pass slots for a pool')
    else:
        N.require(slots.dtype in (torch.int32, torch.int64) and tuple(slots.shape) == (B,),
                  f'slots must be int32 or int64 of shape ({B},) (got {slots.dtype}, {tuple(slots.shape)})')
        slots = slots.contiguous()
    N.require_device(q=q, k=k, v=v, g=g, beta=beta, state=state, slots=slots)
    q, k, v = N.rows_last(q), N.rows_last(k), N.rows_last(v)
    o = torch.empty(B, Hv, V, dtype=v.dtype, device=v.device)
    d = N.SeqDeltaStep(B, state.size(0), Hk, Hv, K, V, N.DTYPES[q.dtype],
                       int(slots is not None and slots.dtype == torch.int64),
                       K ** -0.5 if scale is None else float(scale), q.device.index,
                       q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                       q.stride()[:2], k.stride()[:2], v.stride()[:2], g.stride(), beta.stride(), state.stride()[:2],
                       slots.data_ptr() if slots is not None else None, state.data_ptr(), o.data_ptr())
    N.check(N.load().seq_delta_step(ctypes.byref(d), N.stream(q.device)), 'gated_delta_step')
    return o
