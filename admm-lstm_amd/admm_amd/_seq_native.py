"""Binding of libseqops.so (the C ABI declared in include/seq_ops.h): the sequence-layer operators.

Like libadmmlstm.so (``_native``) it is built in-tree by ``csrc/Makefile`` and is the only compute path of its operators:
loading fails loudly when it is missing, and host tensors are refused.  ``load()`` gives the C ABI through ctypes,
``entry_points()`` the extension ``_seq_torch`` that ``blocks/`` calls.
"""
from __future__ import annotations

import ctypes
import importlib
import os
from ctypes import POINTER, Structure, c_char_p, c_float, c_int, c_int32, c_int64, c_uint64, c_void_p

import torch  # noqa: F401  (must precede the CDLL load: one HIP runtime per process)

from ._native import NativeUnavailable

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'libseqops.so')
ABI_VERSION = 1


class SeqDelta(Structure):
    _fields_ = [('batch', c_int64), ('T', c_int64), ('sequences', c_int64),
                ('Hk', c_int32), ('Hv', c_int32), ('K', c_int32), ('V', c_int32),
                ('dtype', c_int32), ('offsets_64', c_int32), ('scale', c_float), ('device', c_int32),
                ('q', c_void_p), ('k', c_void_p), ('v', c_void_p), ('g', c_void_p), ('beta', c_void_p),
                ('q_stride', c_int64 * 3), ('k_stride', c_int64 * 3), ('v_stride', c_int64 * 3),
                ('g_stride', c_int64 * 3), ('beta_stride', c_int64 * 3),
                ('offsets', c_void_p), ('initial', c_void_p)]


class SeqDeltaStep(Structure):
    _fields_ = [('batch', c_int64), ('pool', c_int64),
                ('Hk', c_int32), ('Hv', c_int32), ('K', c_int32), ('V', c_int32),
                ('dtype', c_int32), ('slots_64', c_int32), ('scale', c_float), ('device', c_int32),
                ('q', c_void_p), ('k', c_void_p), ('v', c_void_p), ('g', c_void_p), ('beta', c_void_p),
                ('q_stride', c_int64 * 2), ('k_stride', c_int64 * 2), ('v_stride', c_int64 * 2),
                ('g_stride', c_int64 * 2), ('beta_stride', c_int64 * 2), ('state_stride', c_int64 * 2),
                ('slots', c_void_p), ('state', c_void_p), ('o', c_void_p)]


class SeqUnit(Structure):
    _fields_ = [('M', c_int64), ('D', c_int32), ('F', c_int32), ('act', c_int32), ('dtype', c_int32), ('device', c_int32),
                ('x', c_void_p), ('wg', c_void_p), ('wu', c_void_p),
                ('x_ld', c_int64), ('wg_ld', c_int64), ('wu_ld', c_int64)]


# name -> (restype, argtypes)
_SIGNATURES = {
    'seq_abi_version': (c_int32, []),
    'seq_last_error': (c_char_p, []),
    'seq_delta_workspace': (c_int, [POINTER(SeqDelta), c_int32, POINTER(c_int64)]),
    'seq_delta_forward': (c_int, [POINTER(SeqDelta), c_int32, c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    'seq_delta_backward_scratch': (c_int, [POINTER(SeqDelta), POINTER(c_int64)]),
    'seq_delta_backward': (c_int, [POINTER(SeqDelta), c_void_p, c_int64, c_void_p, c_int64] + [c_void_p] * 9),
    'seq_delta_step': (c_int, [POINTER(SeqDeltaStep), c_void_p]),
    'seq_dropout': (c_int, [c_int32, c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_uint64, c_uint64, c_void_p, c_int32,
                            c_void_p]),
    'seq_unit_workspace': (c_int, [POINTER(SeqUnit), c_int32, POINTER(c_int64)]),
    'seq_unit_forward': (c_int, [POINTER(SeqUnit), c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    'seq_unit_backward': (c_int, [POINTER(SeqUnit), c_void_p, c_int64, c_void_p, c_void_p, c_int64] + [c_void_p] * 4),
}
EXPORTS = tuple(_SIGNATURES)

_lib = None


def load() -> ctypes.CDLL:
    """Load (once) and return the library, with argtypes/restype declared."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise NativeUnavailable(f'{LIB_PATH} not found: build it with `make -C admm-lstm_amd/admm_amd/csrc` '
                                f'(or __graft_entry__.build()). There is no CPU fallback.')
    try:
        lib = ctypes.CDLL(LIB_PATH)
    except OSError as e:  # pragma: no cover - environment dependent
        raise NativeUnavailable(f'cannot load {LIB_PATH}: {e}') from e
    for name, (res, args) in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    if lib.seq_abi_version() != ABI_VERSION:
        raise NativeUnavailable(f'{LIB_PATH}: ABI {lib.seq_abi_version()} != expected {ABI_VERSION}')
    _lib = lib
    return lib


def entry_points():
    """The extension module with the operators' entry points (csrc/seq_torch.cpp)."""
    load()
    try:
        mod = importlib.import_module('admm_amd._seq_torch')
    except ImportError as e:
        raise NativeUnavailable(f'admm_amd/_seq_torch.so cannot be imported ({e}): build it with '
                                f'`make -C admm-lstm_amd/admm_amd/csrc`. There is no CPU fallback.') from e
    if mod.abi_version() != ABI_VERSION:
        raise NativeUnavailable(f'_seq_torch: ABI {mod.abi_version()} != expected {ABI_VERSION}')
    return mod
