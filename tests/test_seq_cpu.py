"""What the sequence-layer operators refuse, and their C ABI, without a GPU."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_the_header():
    from admm_amd import _seq_native as N
    src = open(os.path.join(ROOT, 'include', 'seq_ops.h')).read()
    names = set(re.findall(r'^(?:int|int32_t|const char\*) (seq_\w+)\(', src, re.M))
    lib = N.load()
    assert names == set(N.EXPORTS)
    for n in names:
        assert hasattr(lib, n)
    assert lib.seq_abi_version() == N.ABI_VERSION


def _delta(**kw):
    from admm_amd import _seq_native as N
    d = N.SeqDelta(batch=2, T=70, sequences=2, Hk=1, Hv=2, K=16, V=24, dtype=0)
    for n, x in kw.items():
        setattr(d, n, x)
    return d


@pytest.mark.parametrize('change, said', [
    (dict(dtype=3), b'dtype'), (dict(Hv=3, Hk=2), b'multiple'), (dict(Hk=0), b'multiple'), (dict(K=129), b'1 to 128'),
    (dict(K=0), b'1 to 128'), (dict(V=0), b'value rows'), (dict(T=-1), b'negative'), (dict(sequences=3), b'sequences'),
    (dict(offsets=64, sequences=5), b'batch 1'), (dict(batch=1 << 40, sequences=1 << 40), b'too many')])
def test_c_abi_refuses_bad_shapes(change, said):
    from admm_amd import _seq_native as N
    lib, n = N.load(), ctypes.c_int64()
    d = _delta(**change)
    assert lib.seq_delta_workspace(ctypes.byref(d), 0, ctypes.byref(n)) == -1
    assert said in lib.seq_last_error()


def test_c_abi_refuses_missing_memory():
    from admm_amd import _seq_native as N
    lib, n = N.load(), ctypes.c_int64()
    d = _delta()
    assert lib.seq_delta_workspace(ctypes.byref(d), 0, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.seq_delta_forward(ctypes.byref(d), 0, None, n.value - 1, None, None, None) == -1
    assert b'work memory' in lib.seq_last_error()
    assert lib.seq_delta_forward(ctypes.byref(d), 0, 256, n.value, None, None, None) == -1
    assert b'NULL' in lib.seq_last_error()
    assert lib.seq_delta_forward(None, 0, None, 0, None, None, None) == -1
    assert lib.seq_delta_step(None, None) == -1
    s = N.SeqDeltaStep(batch=2, pool=1, Hk=1, Hv=1, K=8, V=8, dtype=0)
    assert lib.seq_delta_step(ctypes.byref(s), None) == -1 and b'states' in lib.seq_last_error()


def _rule_args(**kw):
    a = dict(q=torch.zeros(2, 5, 1, 8), k=torch.zeros(2, 5, 1, 8), v=torch.zeros(2, 5, 2, 4), g=torch.zeros(2, 5, 2),
             beta=torch.zeros(2, 5, 2))
    a.update(kw)
    return a


def test_host_tensors_are_refused():
    from blocks.delta_rule import gated_delta_rule, gated_delta_step
    with pytest.raises(RuntimeError, match='HIP device'):
        gated_delta_rule(**_rule_args())
    with pytest.raises(RuntimeError, match='HIP device'):
        gated_delta_step(*(x[:, 0] for x in _rule_args().values()), torch.zeros(2, 2, 8, 4))
    with pytest.raises(TypeError, match='tensor'):
        gated_delta_rule(**_rule_args(q=3))


@pytest.mark.parametrize('change, said', [
    (dict(q=torch.zeros(2, 5, 1, 8).double()), 'q must be'), (dict(k=torch.zeros(2, 5, 1, 8).half()), 'type of q'),
    (dict(g=torch.zeros(2, 5, 2).half()), 'g must be float32'), (dict(beta=torch.zeros(2, 5, 1)), 'beta must have shape'),
    (dict(k=torch.zeros(2, 4, 1, 8)), 'differ in shape'), (dict(v=torch.zeros(2, 4, 2, 4)), 'v has'),
    (dict(v=torch.zeros(2, 5, 4)), 'v must be'), (dict(q=torch.zeros(2, 5, 4, 8), k=torch.zeros(2, 5, 4, 8)), 'multiple'),
    (dict(q=torch.zeros(2, 5, 1, 129), k=torch.zeros(2, 5, 1, 129)), '1 to 128'),
    (dict(q=torch.zeros(2, 5, 1, 0), k=torch.zeros(2, 5, 1, 0)), '1 to 128'),
    (dict(v=torch.zeros(2, 5, 2, 0)), 'empty'),
    (dict(initial_state=torch.zeros(1, 2, 8, 4)), 'initial_state'),
    (dict(initial_state=torch.zeros(2, 2, 8, 4).half()), 'initial_state'),
    (dict(offsets=torch.zeros(2, dtype=torch.int32)), 'batch of 1')])
def test_rule_refusals(change, said):
    from blocks.delta_rule import gated_delta_rule
    with pytest.raises(ValueError, match=said):
        gated_delta_rule(**_rule_args(**change))


@pytest.mark.parametrize('offsets', [torch.zeros(2), torch.zeros(0, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)])
def test_rule_refuses_bad_offsets(offsets):
    from blocks.delta_rule import gated_delta_rule
    one = {n: x[:1] for n, x in _rule_args().items()}
    with pytest.raises(ValueError, match='offsets'):
        gated_delta_rule(**one, offsets=offsets)


@pytest.mark.parametrize('state, slots, said', [
    (torch.zeros(2, 2, 8, 4).half(), None, 'state must'), (torch.zeros(2, 2, 4, 8), None, 'state must'),
    (torch.zeros(3, 2, 8, 4), None, 'pass slots'), (torch.zeros(2, 2, 4, 8).transpose(2, 3), None, 'contiguous'),
    (torch.zeros(1, 2, 8, 4).expand(2, 2, 8, 4), None, 'overlap'), (torch.zeros(2, 1, 8, 4).expand(2, 2, 8, 4), None, 'overlap'),
    (torch.zeros(3, 2, 8, 4), torch.zeros(3, dtype=torch.int32), 'slots'),
    (torch.zeros(3, 2, 8, 4), torch.zeros(2), 'slots')])
def test_step_refusals(state, slots, said):
    from blocks.delta_rule import gated_delta_step
    with pytest.raises(ValueError, match=said):
        gated_delta_step(*(x[:, 0] for x in _rule_args().values()), state, slots=slots)


def test_philox_reference_has_the_published_vectors():
    """Random123's known answers for philox4x32-10: counter and key all zeros, and all ones."""
    import seq_reference as R

    def words(bits):
        return [int(bits[2 * i]) | int(bits[2 * i + 1]) << 16 for i in range(4)]

    assert words(R.philox_bits(8, 0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


@pytest.mark.parametrize('args, kw, said', [
    ((torch.zeros(3, dtype=torch.int32), 0.5, 1), {}, 'x must be'), ((torch.zeros(3), -0.1, 1), {}, 'p must'),
    ((torch.zeros(3), 1.1, 1), {}, 'p must'), ((torch.zeros(3), float('nan'), 1), {}, 'p must'),
    ((torch.zeros(3), 0.5, 1), dict(residual=torch.zeros(4)), 'residual'),
    ((torch.zeros(3), 0.5, 1), dict(residual=torch.zeros(3).half()), 'residual'),
    ((torch.zeros(3), 0.5, torch.zeros(2, dtype=torch.int64)), {}, 'seed'), ((torch.zeros(3), 0.5, torch.zeros(1)), {}, 'seed')])
def test_dropout_refusals(args, kw, said):
    from blocks.dropout import dropout
    with pytest.raises(ValueError, match=said):
        dropout(*args, **kw)


def test_dropout_refuses_host_tensors_and_bad_c_calls():
    from admm_amd import _seq_native as N
    from blocks.dropout import dropout
    with pytest.raises(RuntimeError, match='HIP device'):
        dropout(torch.zeros(3), 0.5, 1)
    lib = N.load()
    assert lib.seq_dropout(5, 1, None, 1, 4, 0, 0, 0, None, 0, None) == -1
    assert lib.seq_dropout(0, 1, None, 1, -4, 0, 0, 0, None, 0, None) == -1
    assert lib.seq_dropout(0, 1, None, 1, 4, 65537, 0, 0, None, 0, None) == -1
    assert lib.seq_dropout(0, None, None, 1, 4, 0, 0, 0, None, 0, None) == -1
    assert lib.seq_dropout(0, None, None, None, 0, 0, 0, 0, None, 0, None) == 0


@pytest.mark.parametrize('x, wg, wu, kw, said', [
    (torch.zeros(2, 4).double(), torch.zeros(4, 3).double(), torch.zeros(4, 3).double(), {}, 'x must be'),
    (torch.zeros(2, 4), torch.zeros(4, 3).half(), torch.zeros(4, 3), {}, 'w_gate must have'),
    (torch.zeros(2, 4), torch.zeros(5, 3), torch.zeros(4, 3), {}, 'w_gate must be'),
    (torch.zeros(2, 4), torch.zeros(4, 3), torch.zeros(4), {}, 'w_up must be'),
    (torch.zeros(2, 4), torch.zeros(4, 3), torch.zeros(4, 2), {}, 'differ in shape'),
    (torch.zeros(2, 4), torch.zeros(4, 0), torch.zeros(4, 0), {}, 'between 1 x 1'),
    (torch.zeros(2, 0), torch.zeros(0, 3), torch.zeros(0, 3), {}, 'between 1 x 1'),
    (torch.zeros(()), torch.zeros(4, 3), torch.zeros(4, 3), {}, 'one axis'),
    (torch.zeros(2, 4), torch.zeros(4, 3), torch.zeros(4, 3), dict(activation='relu'), 'activation')])
def test_unit_refusals(x, wg, wu, kw, said):
    from blocks.gated_unit import gated_unit
    with pytest.raises(ValueError, match=said):
        gated_unit(x, wg, wu, **kw)


def test_unit_refuses_host_tensors_and_bad_c_calls():
    from admm_amd import _seq_native as N
    from blocks.gated_unit import gated_unit
    with pytest.raises(RuntimeError, match='HIP device'):
        gated_unit(torch.zeros(2, 4), torch.zeros(4, 3), torch.zeros(4, 3))
    lib, n = N.load(), ctypes.c_int64()

    def bad(said, **kw):
        u = N.SeqUnit(M=4, D=8, F=8, x_ld=8, wg_ld=8, wu_ld=8)
        for name, v in kw.items():
            setattr(u, name, v)
        assert lib.seq_unit_workspace(ctypes.byref(u), 0, ctypes.byref(n)) == -1 and said in lib.seq_last_error()

    bad(b'dtype', dtype=7)
    bad(b'activation', act=3)
    bad(b'rows', M=-1)
    bad(b'weights', D=0)
    bad(b'weights', F=(1 << 20) + 1)
    bad(b'too many', M=(1 << 31) - 1, F=1 << 20)
    u = N.SeqUnit(M=40, D=7, F=7, x_ld=7, wg_ld=7, wu_ld=7)   # (up to 32 rows need no work memory)
    assert lib.seq_unit_workspace(ctypes.byref(u), 1, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.seq_unit_forward(ctypes.byref(u), None, 0, None, None, None) == -1 and b'work memory' in lib.seq_last_error()
    assert lib.seq_unit_backward(ctypes.byref(u), 256, n.value, None, None, 7, None, None, None, None) == -1


def test_lstm_dropout_refusals_and_default():
    from blocks.lstm import LSTM
    for kw, said in ((dict(with_grad=True, dropout=1.5), 'between 0 and 1'), (dict(dropout=0.5), 'with_grad')):
        with pytest.raises(ValueError, match=said):
            LSTM(3, 4, 1, **kw)
    torch.manual_seed(0)
    a = LSTM(3, 4, 1, with_grad=True)
    torch.manual_seed(0)
    b = LSTM(3, 4, 1, with_grad=True, dropout=0.5).eval()
    x = torch.randn(2, 5, 3)
    assert torch.equal(a(x), b(x)) and list(a.state_dict()) == list(b.state_dict())
