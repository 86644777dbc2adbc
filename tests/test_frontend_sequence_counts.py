"""lengths and top_k of the sequence operators as the host gives them: integers of any width, nothing else."""
import ctypes as C

import numpy as np
import pytest

import charmnumeric_amd as cnp
from charmnumeric_amd import _lib as L
from charmnumeric_amd import lazy


@pytest.fixture
def itf():
    cnp.reset()
    it = cnp.CharmNumericInterface(device=-1)
    it.connect(odf=4)
    it.set_trace()
    yield it
    cnp.reset()
    it.close()


def f32(*shape):
    return cnp.array(np.arange(1, np.prod(shape) + 1, dtype=np.float32).reshape(shape))


def uploaded(call):
    """What `call` uploads: the arrays of the put calls it records."""
    before = len(lazy._state.pending)
    call()
    return [r.payload for r in lazy._state.pending[before:] if not isinstance(r, bytes) and r.opcode == "put"]


@pytest.mark.parametrize("given", [
    [2.7, 1.2], [2.0, 1.0], (1.5, 2), np.array([2.7, 1.2]), np.array([2, 1], np.float32), [float("nan"), 1.0], ["2", "1"],
    [1 + 0j, 2],
])
def test_what_is_no_integer_is_refused(itf, given):
    x, w, logits = f32(2, 5, 8), f32(4, 8), f32(2, 50)
    with pytest.raises(TypeError):
        cnp.short_convolution(x, w, lengths=given)
    with pytest.raises(TypeError):
        cnp.state_scan(x, x, f32(8, 4), f32(2, 5, 4), f32(2, 5, 4), lengths=given)
    if not any(isinstance(v, str) for v in given):
        with pytest.raises(TypeError):
            cnp.random.sample_tokens(logits, np.array([0.1, 0.2]), top_k=given)


@pytest.mark.parametrize("given,want", [
    (np.array([2 ** 32 + 3, -2 ** 40], np.int64), [2 ** 31 - 1, -2 ** 31]),
    (np.array([2 ** 63 + 5, 3], np.uint64), [2 ** 31 - 1, 3]),
    ([2 ** 31, 4], [2 ** 31 - 1, 4]),
    (np.array([3, -1], np.int8), [3, -1]),
    ([5, 2], [5, 2]),
])
def test_integers_of_any_width_are_held_to_32_bits(itf, given, want):
    x, w, logits = f32(2, 5, 8), f32(4, 8), f32(2, 50)
    u = cnp.array(np.array([0.1, 0.2]))
    for call in (lambda: cnp.short_convolution(x, w, lengths=given), lambda: cnp.random.sample_tokens(logits, u, top_k=given)):
        put = uploaded(call)
        assert len(put) == 1 and put[0].dtype == np.int32 and put[0].tolist() == want


def test_arrays_of_64_bits_go_to_the_executor_as_they_are(itf):
    """Their values are not known here: the executor holds them to 32 bits on the device, in a buffer of the call."""
    x, w, logits = f32(2, 5, 8), f32(4, 8), f32(2, 50)
    u, n = cnp.array(np.array([0.1, 0.2])), cnp.array(np.array([2, 2 ** 40]))
    calls = [cnp.short_convolution(x, w, lengths=n), cnp.random.sample_tokens(logits, u, top_k=n),
             cnp.state_scan(x, x, f32(8, 4), f32(2, 5, 4), f32(2, 5, 4), lengths=n)]
    cnp.execute(itf)
    itf.sync()
    log = itf.trace()
    assert sum(ln.startswith("narrow %d " % n.name) for ln in log) == 3
    assert not any(ln.startswith("astype") for ln in log)
    del calls
    with pytest.raises(L.CnhError):                           # as before: of the right extents only
        bad = cnp.array(np.array([1, 2, 3]))
        whole = L.Operand(x.name, L.Region.make())
        L.check(L.lib.cnx_short_convolution(itf._ex, C.byref(L.XShortConvolution(whole, w.name, 0, 0, bad.name, 901, 1))))
