"""Dropout whose mask is never stored.

``y = residual + x * keep / P(keep)``, where ``keep`` of element i (counted over the contiguous tensor) comes from
Philox4x32-10 at counter (i // 8, offset) under the key ``seed``, 16 bits an element: it is dropped where those are below
``round(65536 * p)``.  So p takes steps of 1/65536, the same seed and offset give the same mask on any launch, and the
backward pass recomputes it.  Runs in libseqops.so (a hand-written gfx950 kernel) on the current stream.
"""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from admm_amd import _seq_native as N


def _run(x, residual, below, seed, offset):
    y = torch.empty_like(x)
    on_device = isinstance(seed, torch.Tensor)
    N.check(N.load().seq_dropout(N.DTYPES[x.dtype], x.data_ptr(), residual.data_ptr() if residual is not None else None,
                                 y.data_ptr(), x.numel(), below, 0 if on_device else seed, offset,
                                 seed.data_ptr() if on_device else None, x.device.index, N.stream(x.device)), 'dropout')
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, below, seed, offset):
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)   # an edit between the passes is an error, not another mask
        else:
            ctx.seed = seed
        ctx.below, ctx.offset = below, offset
        return _run(x, residual, below, seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        seed = ctx.saved_tensors[0] if ctx.saved_tensors else ctx.seed
        dx = _run(dy.contiguous(), None, ctx.below, seed, ctx.offset) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], *, offset: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` with each element dropped with probability ``p`` and the kept ones divided by 1 - p, plus ``residual``.

    x (bfloat16, float16 or float32) and residual have the same shape and type; the result is contiguous.  A dropped
    element counts as zero whatever it holds (NaN too); p = 1 drops all.  ``seed`` is an integer, or one int64 value on the
    device, read when the kernel runs: a captured call then draws a new mask each time that value is changed.  ``offset``
    tells calls under one seed apart (layers, steps).  Gradients reach x and residual.
    """
    N.require_tensors(x=x, residual=residual)
    N.require(x.dtype in N.DTYPES, f'x must be bfloat16, float16 or float32 (got {x.dtype})')
    N.require(0.0 <= p <= 1.0, f'p must be between 0 and 1 (got {p})')
    if residual is not None:
        N.require(residual.shape == x.shape and residual.dtype == x.dtype,
                  f'residual must be {x.dtype} of shape {tuple(x.shape)} (got {residual.dtype}, {tuple(residual.shape)})')
    if isinstance(seed, torch.Tensor):
        N.require(seed.dtype == torch.int64 and seed.numel() == 1,
                  f'seed must be an integer or one int64 value (got {seed.dtype}, shape {tuple(seed.shape)})')
        N.require_device(x=x, residual=residual, seed=seed)
    else:
        seed = int(seed) & 0xffffffffffffffff
        N.require_device(x=x, residual=residual)
    offset = int(offset) & 0xffffffffffffffff
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    below = int(round(p * 65536))
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, below, seed, offset)
    return _run(x, residual, below, seed, offset)
