"""The sequence operators of the frontend without a device: checks of arguments, what is recorded, and the
decisions of the executor's dry mode."""
import numpy as np
import pytest

import charmnumeric_amd as cnp
from charmnumeric_amd import _lib as L


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


def lines(itf, *prefixes):
    cnp.execute(itf)
    itf.sync()
    return [ln for ln in itf.trace() if ln.startswith(prefixes)]


def test_refusals_of_the_functions(itf):
    x, w, A = f32(2, 5, 8), f32(4, 8), f32(8, 16)
    B = f32(2, 5, 16)
    st = cnp.zeros((2, 8, 16), dtype=np.float32)
    cs = cnp.zeros((2, 3, 8), dtype=np.float32)
    logits, u = f32(3, 50), cnp.random.uniform((3,), 1)
    scan = lambda **k: cnp.state_scan(**{**dict(x=x, delta=x, A=A, B=B, C=B), **k})  # noqa: E731
    bad = [
        (ValueError, lambda: cnp.rms_norm(x, eps=-1.0)),
        (ValueError, lambda: cnp.rms_norm(x, eps=float("nan"))),
        (ValueError, lambda: cnp.rms_norm(x, f32(7))),
        (ValueError, lambda: cnp.rms_norm(x, residual=cnp.zeros((2, 5, 7), dtype=np.float32))),
        (TypeError, lambda: cnp.rms_norm(x, residual=np.zeros((2, 5, 8), np.float32))),
        (TypeError, lambda: cnp.rms_norm(x.astype(np.float64), residual=cnp.zeros((2, 5, 8), dtype=np.float32))),
        (ValueError, lambda: cnp.rms_norm(x, residual=x)),
        (ValueError, lambda: cnp.rms_norm(x[:1], residual=x)),
        (ValueError, lambda: cnp.rms_norm(x[:, 1:], residual=x[:, :4])),
        (TypeError, lambda: cnp.rms_norm(3.0)),
        (ValueError, lambda: cnp.short_convolution(f32(8), w)),
        (ValueError, lambda: cnp.short_convolution(x, f32(9, 8))),
        (ValueError, lambda: cnp.short_convolution(x, f32(4, 7))),
        (ValueError, lambda: cnp.short_convolution(x, w, activation="relu")),
        (ValueError, lambda: cnp.short_convolution(x, w, state=cnp.zeros((2, 4, 8), dtype=np.float32))),
        (ValueError, lambda: cnp.short_convolution(x, f32(1, 8), state=cs)),
        (TypeError, lambda: cnp.short_convolution(x, w, lengths=x[:, 0, 0])),
        (ValueError, lambda: cnp.short_convolution(x, w, lengths=[1, 2, 3])),
        (ValueError, lambda: cnp.short_convolution(x, w, bias=f32(9))),
        (ValueError, lambda: scan(A=f32(7, 16))),
        (ValueError, lambda: scan(A=f32(8, 257))),
        (ValueError, lambda: scan(B=f32(2, 5, 15))),
        (ValueError, lambda: scan(C=f32(2, 4, 16))),
        (ValueError, lambda: scan(C=None)),
        (ValueError, lambda: scan(z=f32(2, 5, 9))),
        (ValueError, lambda: scan(skip=f32(9))),
        (ValueError, lambda: scan(state=st[:, :, :8])),
        (ValueError, lambda: scan(state=cnp.zeros((2, 8, 15), dtype=np.float32))),
        (TypeError, lambda: scan(state=cnp.zeros((2, 8, 16), dtype=np.int32))),
        (ValueError, lambda: cnp.random.sample_tokens(f32(2, 3, 4), u)),
        (ValueError, lambda: cnp.random.sample_tokens(logits, cnp.random.uniform((4,), 1))),
        (ValueError, lambda: cnp.random.sample_tokens(logits, u, temperature=-1.0)),
        (ValueError, lambda: cnp.random.sample_tokens(logits, u, temperature=float("nan"))),
        (ValueError, lambda: cnp.random.sample_tokens(logits, u, top_k=-1)),
        (TypeError, lambda: cnp.random.sample_tokens(logits, u, top_k=1.5)),
        (TypeError, lambda: cnp.random.sample_tokens(logits, u, top_k=np.ones(3))),
        (ValueError, lambda: cnp.random.sample_tokens(logits, u, min_p=1.5)),
        (ValueError, lambda: cnp.random.sample_tokens(logits, u, top_p=np.ones(4))),
    ]
    cnp.execute(itf)
    itf.trace()
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            raise AssertionError(f"call {i} was taken")
    assert lines(itf, "rms_norm", "short_conv", "state_scan", "sample") == []


def test_program_order_and_names(itf):
    """A call stands behind the statements recorded before it and in front of those after it, and its
    result is deleted when its handle goes."""
    x = f32(2, 5, 8)
    y = x * 2.0
    n = cnp.rms_norm(y)
    z = n + y
    del n
    got = lines(itf, "group", "rms_norm", "dense", "delete", "create")
    at = [i for i, ln in enumerate(got) if ln.startswith("rms_norm")]
    assert len(at) == 1
    before, after = got[:at[0]], got[at[0]:]
    assert any(ln.startswith("create %d " % y.name) for ln in before)
    assert any(ln.startswith("create %d " % z.name) for ln in after)
    assert any(ln.startswith("delete") for ln in after)
    info = itf.array_info(z.name)
    assert info["shape"] == (2, 5, 8) and info["dtype"] == L.F32


def test_types_meet_in_the_result_type(itf):
    x = f32(2, 5, 8)
    assert cnp.rms_norm(x).dtype == np.float32
    assert cnp.rms_norm(x, np.ones(8)).dtype == np.float64
    assert cnp.rms_norm(cnp.array(np.arange(6).reshape(2, 3))).dtype == np.float64
    assert cnp.short_convolution(x, np.ones((4, 8), np.float32)).dtype == np.float32
    assert cnp.random.sample_tokens(f32(3, 9), np.array([0.1, 0.2, 0.3])).dtype == np.int32
    assert cnp.random.sample_tokens(f32(9), np.array([0.5], np.float32), top_k=np.array([3])).shape == (1,)
    cnp.execute(itf)
    itf.sync()


def test_slices_are_read_in_place_where_they_can_be(itf):
    x = f32(4, 6, 16)
    w = f32(4, 8)
    cnp.execute(itf)
    itf.trace()
    ys = [cnp.short_convolution(x[:, :, 8:], w), cnp.short_convolution(x[1:3, 2:, :8], w), cnp.rms_norm(x[:, :, 4:12])]
    assert len(lines(itf, "create")) == 3                     # the results alone
    ys += [cnp.short_convolution(x[:, ::2, :8], w), cnp.rms_norm(x[:, 1:, :])]
    assert len(lines(itf, "create")) == 4                     # a copy each
    assert ys[1].shape == (2, 4, 8)


def test_the_executor_refuses_what_does_not_fit(itf):
    """The C entry points check for themselves: operands that are not there, regions, extents."""
    x = f32(2, 5, 8)
    n = f32(8)
    cnp.execute(itf)
    import ctypes as C
    whole = L.Operand(x.name, L.Region.make())
    call = lambda **k: L.lib.cnx_rms_norm(itf._ex, C.byref(L.XRmsNorm(**{**dict(x=whole, y=900, eps=1e-6), **k})))  # noqa: E731
    assert call() == 0
    assert call() < 0 and "already exists" in L.lib.cnh_last_error().decode()
    assert call(y=901, x=L.Operand(77, L.Region.make())) < 0
    assert call(y=901, weight=x.name) == -50
    assert call(y=901, residual=n.name) == -50
    assert call(y=901, x=L.Operand(x.name, L.Region.make((0, 0, 0), (2, 5, 9), (1, 1, 1)))) == -50
    assert call(y=901, x=L.Operand(x.name, L.Region.make((0, 0, 0), (2, 5, 8), (1, 2, 1)))) == -50
    assert call(y=901, x=L.Operand(x.name, L.Region.make((0, 1, 0), (2, 5, 8), (1, 1, 1)))) == -50
    assert call(y=901, x=L.Operand(x.name, L.Region.make((0, 1, 0), (1, 5, 8), (1, 1, 1)))) == 0


def test_struct_layouts_match_the_header(tmp_path):
    import ctypes as C
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"cnx_operand": L.Operand, "cnx_rms_norm_args": L.XRmsNorm, "cnx_short_convolution_args": L.XShortConvolution,
               "cnx_state_scan_args": L.XStateScan, "cnx_sample_tokens_args": L.XSampleTokens}
    lines_ = []
    for name, cls in structs.items():
        lines_.append(f'printf("%zu\\n", sizeof({name}));')
        lines_ += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "cnexec.h"\nint main(void) {\n' + "\n".join(lines_) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I" + os.path.join(root, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    want = []
    for cls in structs.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want
