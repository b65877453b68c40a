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


def _unit(M, F, D=8, dtype=0, backward=0):
    from admm_amd import _seq_native as N
    return _size('seq_unit_workspace', N.SeqUnit(M=M, D=D, F=F, dtype=dtype, x=16, wg=16, wu=16, x_ld=D, wg_ld=F, wu_ld=F), backward)


def test_launches_of_the_unit():
    rc, said = _unit((1 << 31) - 256, 8)   # tiles of 64 rows with 256 threads each, or fewer with 512
    assert rc == -1 and b'too many rows' in said
    assert _unit((1 << 30) - 256, 8)[0] == 0
    assert _unit(1 << 22, 8192)[0] == 0 and _unit(1 << 22, 8192, backward=1)[0] == 0   # 2^20 tiles of 512 threads
    rc, said = _unit(1 << 26, 1 << 14)   # 2^25 tiles of 512 threads
    assert rc == -1 and b'too many rows' in said
    rc, said = _unit(1 << 26, 8, D=1 << 15, backward=1)   # the gradient of x alone is too large
    assert rc == -1 and b'too many rows' in said


def _delta(N, B, T, H, K=1, V=1, dtype=0):
    return N.SeqDelta(batch=B, T=T, sequences=B, Hk=H, Hv=H, K=K, V=V, dtype=dtype)


@pytest.mark.parametrize('saved', [0, 1])
def test_launches_of_the_rule(saved):
    """A workgroup of 256 threads a sequence and head up to 32 rows; 512 threads a column tile of a longer one (256 in chunks of 32
    rows)."""
    from admm_amd import _seq_native as N

    def ask(*a, **kw):
        return _size('seq_delta_workspace', _delta(N, *a, **kw), saved)

    most = (THREADS - 1) // 256
    assert ask(most, 4, 1)[0] == 0 and ask(most // 4, 4, 4)[0] == 0
    for a in ((most + 1, 4, 1), (most // 4 + 1, 4, 4), (1 << 31, 4, 1)):
        rc, said = ask(*a)
        assert rc == -1 and b'too many' in said, a
    rc, said = ask(THREADS // 512 + 8, 65, 1, K=64, V=32)   # one workgroup of two tiles each, in chunks of 32 rows or (saved) of 64
    assert rc == -saved and (not saved or b'too many' in said)


def test_launches_of_single_tokens():
    """256 threads for 32 columns of a head's state, or for 128 of them."""
    from admm_amd import _seq_native as N

    def ask(B, V):
        d = N.SeqDeltaStep(batch=B, pool=B, Hk=1, Hv=1, K=1, V=V, dtype=0, device=0)   # no buffers: nothing is launched
        return N.load().seq_delta_step(ctypes.byref(d), None), N.load().seq_last_error()

    most = (THREADS - 1) // 256
    for B, V, fits in ((most, 32, True), (most + 1, 32, False), (most // 2, 33, True), (most // 2 + 1, 33, False),
                       (most, 128, True), (most + 1, 128, False)):
        rc, said = ask(B, V)
        assert rc == -1 and (b'NULL' in said if fits else b'too many' in said), (B, V, said)
