"""Dropout whose mask is never stored.

``y = residual + x * keep / P(keep)``, where ``keep`` of element i (counted over the contiguous tensor) comes from
Philox4x32-10 at counter (i // 8, offset) under the key ``seed``, 16 bits an element: it is dropped where those are below
``round(65536 * p)``.  So p takes steps of 1/65536, the same seed and offset give the same mask on any launch, and the
backward pass recomputes it.  Runs in libseqops.so (a hand-written gfx950 kernel) on the current stream.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from admm_amd import _seq_native

_E = _seq_native.entry_points()


def dropout(x: torch.Tensor, p: float, seed: Union[int, torch.Tensor], *, offset: int = 0,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` with each element dropped with probability ``p`` and the kept ones divided by 1 - p, plus ``residual``.

    x (bfloat16, float16 or float32) and residual have the same shape and type; the result is contiguous.  A dropped
    element counts as zero whatever it holds (NaN too); p = 1 drops all.  ``seed`` is an integer, or one int64 value on the
    device, read when the kernel runs: a captured call then draws a new mask each time that value is changed.  ``offset``
    tells calls under one seed apart (layers, steps).  Gradients reach x and residual.
    """
    return _E.dropout(x, p, seed, offset, residual)
