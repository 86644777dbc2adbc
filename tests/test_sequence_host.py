"""The sequence operators' C entry points without a device: layouts, workspaces, refusals."""
import ctypes as C
import os
import subprocess

import pytest

from charmnumeric_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"cnh_rms_norm_args": L.RmsNorm, "cnh_short_convolution_args": L.ShortConvolution,
           "cnh_state_scan_args": L.StateScan, "cnh_sample_tokens_args": L.SampleTokens}
BIG = 1 << 30


def test_layouts_match_the_header(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cnhip.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    want = []
    for cls in STRUCTS.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def norm(**kw):
    a = L.RmsNorm(L.F32, 4, 8, 1 * BIG, 8, 2 * BIG, 8, 3 * BIG, 8, 4 * BIG, 1e-6, 5 * BIG, 8)
    return set_all(a, kw)


def conv(**kw):
    a = L.ShortConvolution(L.F32, 1, 4, 2, 5, 8, 1 * BIG, 40, 8, 2 * BIG, 3 * BIG, 4 * BIG, 5 * BIG, 6 * BIG,
                           7 * BIG, 40, 8)
    return set_all(a, kw)


def scan(**kw):
    a = L.StateScan(L.F32, 1, 2, 5, 8, 16, 1 * BIG, 40, 8, 2 * BIG, 40, 8, 3 * BIG, 40, 8, 4 * BIG, 5 * BIG, 80, 16,
                    6 * BIG, 80, 16, 7 * BIG, 8 * BIG, 9 * BIG, 10 * BIG, 11 * BIG, 12 * BIG, 40, 8, None, 0)
    return set_all(a, kw)


def sample(**kw):
    a = L.SampleTokens(L.F32, 0, 3, 100, 1 * BIG, 100, 2 * BIG, 1.0, 1.0, 0.0, None, None, None, None, 3 * BIG, None, 0)
    return set_all(a, kw)


def set_all(a, kw):
    for k, v in kw.items():
        assert hasattr(a, k), k
        setattr(a, k, v)
    return a


CALLS = {norm: L.lib.cnh_rms_norm, conv: L.lib.cnh_short_convolution, scan: L.lib.cnh_state_scan,
         sample: L.lib.cnh_sample_tokens}
NAN = float("nan")


@pytest.mark.parametrize("make,kw,rc,word", [
    (norm, dict(dtype=L.I32), -2, "element type"),
    (norm, dict(rows=-1), -2, "rows"),
    (norm, dict(rows=1 << 31), -3, "below"),
    (norm, dict(x=None), -2, "null"),
    (norm, dict(y=None), -2, "null"),
    (norm, dict(eps=NAN), -2, "eps"),
    (norm, dict(eps=-1.0), -2, "eps"),
    (norm, dict(residual=None), -2, "without a residual"),
    (norm, dict(x_stride=-8), -2, "stride of x"),
    (norm, dict(y_stride=7), -2, "rows of an output"),
    (norm, dict(residual_out_stride=0), -2, "rows of an output"),
    (norm, dict(y=1 * BIG + 124), -2, "y overlaps x"),
    (norm, dict(y=2 * BIG), -2, "y overlaps residual"),
    (norm, dict(residual_out=1 * BIG), -2, "overlaps x or weight"),
    (norm, dict(residual_out=2 * BIG + 32), -2, "without being the same"),
    (norm, dict(residual_out=2 * BIG, residual_stride=9, residual_out_stride=8), -2, "without being the same"),
    (norm, dict(x=BIG + 2), -2, "not aligned"),
    (conv, dict(dtype=7), -2, "element type"),
    (conv, dict(taps=0), -3, "taps"),
    (conv, dict(taps=9), -3, "taps"),
    (conv, dict(activation=2), -2, "activation"),
    (conv, dict(length=-5), -2, "length"),
    (conv, dict(weight=None), -2, "null"),
    (conv, dict(y=None), -2, "null"),
    (conv, dict(x_stride=-1), -2, "stride of x"),
    (conv, dict(y_stride=4), -2, "rows of y"),
    (conv, dict(y_batch_stride=39), -2, "rows of y"),
    (conv, dict(y=1 * BIG), -2, "y overlaps x"),
    (conv, dict(y=5 * BIG), -2, "y overlaps state_out"),
    (conv, dict(state_out=4 * BIG + 32), -2, "without being the same"),
    (conv, dict(state_out=6 * BIG), -2, "state_out overlaps lengths"),
    (conv, dict(lengths=6 * BIG + 2), -2, "not aligned"),
    (conv, dict(channels=1 << 28), -3, "channels"),
    (conv, dict(length=1 << 31), -3, "length"),
    (scan, dict(dtype=L.I64), -2, "element type"),
    (scan, dict(states=0), -3, "states"),
    (scan, dict(states=257), -3, "states"),
    (scan, dict(softplus=3), -2, "softplus"),
    (scan, dict(batch=-1), -2, "batch"),
    (scan, dict(channels=1 << 24), -3, "channels"),
    (scan, dict(batch=1, length=2, x=100 * BIG, x_stride=1 << 29), -3, "less than 2 GiB"),
    (scan, dict(batch=1, length=2, C=100 * BIG, C_stride=1 << 29), -3, "less than 2 GiB"),
    (scan, dict(dtype=L.F64, batch=1, length=2, y=100 * BIG, y_stride=1 << 28), -3, "less than 2 GiB"),
    (scan, dict(A=None), -2, "null"),
    (scan, dict(delta=None), -2, "null"),
    (scan, dict(B_stride=-1), -2, "stride of B"),
    (scan, dict(y_stride=7), -2, "rows of y"),
    (scan, dict(y=2 * BIG), -2, "y overlaps delta"),
    (scan, dict(state_out=4 * BIG), -2, "state_out overlaps A"),
    (scan, dict(state_out=9 * BIG + 64, state_in=9 * BIG), -2, "without being the same"),
    (scan, dict(length=4096, x_batch_stride=1 << 15, delta_batch_stride=1 << 15, z_batch_stride=1 << 15,
                B_batch_stride=1 << 16, C_batch_stride=1 << 16, y_batch_stride=1 << 15), -2, "workspace of"),
    (sample, dict(dtype=L.I32), -2, "element type"),
    (sample, dict(vocab=1 << 17, stride=1 << 17, u=10 * BIG, out=11 * BIG), -2, "workspace of"),
    (sample, dict(vocab=1 << 17, stride=1 << 17, u=10 * BIG, out=11 * BIG, workspace=12 * BIG, workspace_bytes=9), -2,
     "workspace of"),
    (sample, dict(vocab=1 << 17, stride=1 << 17, u=10 * BIG, out=11 * BIG, workspace=10 * BIG, workspace_bytes=BIG), -2,
     "workspace overlaps u"),
    (sample, dict(vocab=0), -3, "words"),
    (sample, dict(vocab=(1 << 22) + 1), -3, "words"),
    (sample, dict(rows=-1), -3, "rows"),
    (sample, dict(temperature=-0.5), -2, "temperature"),
    (sample, dict(temperature=NAN), -2, "temperature"),
    (sample, dict(top_k=-1), -2, "top_k"),
    (sample, dict(top_p=NAN), -2, "top_p"),
    (sample, dict(min_p=1.5), -2, "min_p"),
    (sample, dict(u=None), -2, "null"),
    (sample, dict(out=1 * BIG + 4), -2, "out overlaps"),
    (sample, dict(out=2 * BIG), -2, "out overlaps u"),
    (sample, dict(stride=-100), -2, "stride of logits"),
    (sample, dict(u=2 * BIG + 4), -2, "not aligned"),
])
def test_refusals(make, kw, rc, word):
    got = CALLS[make](C.byref(make(**kw)), None)
    text = L.lib.cnh_last_error().decode()
    assert got == rc and word in text, (got, text)


def test_null_arguments():
    for call in CALLS.values():
        assert call(None, None) == -2
    assert L.lib.cnh_state_scan_workspace(None) == -2
    assert L.lib.cnh_sample_tokens_workspace(None) == -2


def test_no_work_needs_no_device():
    for make, kw in ((norm, dict(rows=0, x=None, y=None)), (norm, dict(cols=0)), (conv, dict(batch=0)),
                     (conv, dict(length=0, state_out=None, x=None, y=None)), (scan, dict(channels=0)),
                     (scan, dict(length=0, state_out=None, x=None, y=None)), (sample, dict(rows=0, logits=None))):
        assert CALLS[make](C.byref(make(**kw)), None) == 0, (make, kw, L.lib.cnh_last_error())


def test_workspaces():
    need = lambda **kw: L.lib.cnh_state_scan_workspace(C.byref(scan(**kw)))  # noqa: E731
    assert need(length=1, batch=64, channels=4096) == 0
    assert need(length=0) == 0
    assert need(batch=64, channels=4096, length=4096) == 0        # fills the device by itself
    one = need(batch=1, channels=2048, length=8192)
    # pieces x (states + 1) x channels of 4 bytes
    assert one > 0 and one % (17 * 2048 * 4) == 0
    assert need(batch=1, channels=2048, length=8192, dtype=L.F64) == 2 * one
    assert need(states=500) == -3
    words = lambda **kw: L.lib.cnh_sample_tokens_workspace(C.byref(sample(**kw)))  # noqa: E731
    assert words() == 0
    # a histogram of 2048 masses and counts, the mass above min-p and the slices' maxima for each row
    assert words(rows=2, vocab=131072, stride=131072) == 2 * (2048 * 12 + 8 + 16 * 4)
    assert words(rows=2, vocab=131072, top_k=50) == 0 and words(rows=2, vocab=131072, temperature=0.0) == 0
    assert words(rows=2, vocab=131072, top_k=50, top_ks=BIG * 9) > 0
    assert words(rows=200, vocab=131072) == 0 and words(vocab=-1) == -3
