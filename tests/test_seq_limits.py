"""The largest calls of the sequence-layer operators, by their C ABI and without a GPU: what no launch can hold is refused before
anything is enqueued, and what one can hold is not."""
import ctypes

import pytest

THREADS = 1 << 32   # a launch takes fewer threads than this along an axis


def _size(call, d, flag):
    from admm_amd import _seq_native as N
    n = ctypes.c_int64()
    rc = getattr(N.load(), call)(ctypes.byref(d), flag, ctypes.byref(n))
    return rc, N.load().seq_last_error()


@pytest.mark.parametrize('backward', [0, 1])
@pytest.mark.parametrize('dtype', [0, 1, 2])
def test_rows_of_the_unit(backward, dtype):
    """Row numbers, and those of the last tile, are 32-bit integers."""
    from admm_amd import _seq_native as N

    def ask(M):
        return _size('seq_unit_workspace', N.SeqUnit(M=M, D=8, F=8, dtype=dtype, x=16, wg=16, wu=16, x_ld=8, wg_ld=8, wu_ld=8), backward)

    for M in ((1 << 31) - 1, (1 << 31) - 255, 1 << 31, 1 << 40):
        rc, said = ask(M)
        assert rc == -1 and b'rows' in said, M
    assert ask((1 << 30) - 256)[0] == 0
