"""Native (gfx950 HIP) implementation behind the admm-lstm_amd drop-in modules.

Layout of the drop-in directory (put ``admm-lstm_amd/`` on ``sys.path``, as the
reference's own directory is when ``demo.py`` runs):

* ``admm.py`` / ``admm.no_dual_y.py`` -- ``ADMMBasedOptimizer`` (both variants)
* ``blocks/lstm.py`` -- ``LSTM`` model container
* ``blocks/delta_rule.py``, ``blocks/gated_unit.py``, ``blocks/dropout.py`` -- operators of sequence
  layers for PyTorch, forward and backward: the gated delta rule (whole sequences and single tokens),
  the gated unit, dropout without a stored mask
* ``parameters.py`` -- rho/beta dictionaries
* ``_global.py`` -- device and message/exit conventions
* ``admm_amd/`` -- ctypes binding (``_native``), host logic (``optimizer``), HIP sources
  (``csrc/``) and the built ``libadmmlstm.so``; ``_seq_native`` loads ``libseqops.so`` (C ABI in
  ``include/seq_ops.h``) and ``_seq_torch.so``, its entry points for PyTorch
"""
from . import _native  # noqa: F401

__all__ = ['_native']
