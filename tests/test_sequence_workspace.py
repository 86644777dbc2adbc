"""How much workspace the draw asks for, by its settings."""
import ctypes as C
import itertools

import pytest

from charmnumeric_amd import _lib as L

BIG = 1 << 30


@pytest.mark.parametrize("dtype", [L.F32, L.F64])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 16383), (1, 16384), (1, 131072), (3, 50021), (16, 131072), (17, 131072),
                                        (128, 131072), (129, 1 << 22), (1, 1 << 22)])
def test_one_workspace_for_all_settings(dtype, rows, vocab):
    """top_k 0 and temperature 1 ask for the most; the number changes with the settings, as the header says."""
    def need(top_k, temperature, per_row_k, per_row_t):
        a = L.SampleTokens(dtype, top_k, rows, vocab, 1 * BIG, vocab, 2 * BIG, temperature, 0.9, 0.1)
        a.top_ks, a.temperatures = 3 * BIG if per_row_k else None, 4 * BIG if per_row_t else None
        return L.check(L.lib.cnh_sample_tokens_workspace(C.byref(a)))
    most = need(0, 1.0, False, False)
    every = {need(*q) for q in itertools.product((0, 1, 50, 512, 513, vocab), (0.0, 0.7, 1.0), (False, True), (False, True))}
    assert max(every) == most and every <= {0, most}
    assert need(50, 1.0, False, False) == 0 and need(0, 0.0, False, False) == 0
