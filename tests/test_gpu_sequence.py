"""The sequence operators on the device through the C entry points, against their definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from charmnumeric_amd import _lib as L
from tests import helpers as H
from tests import sequence_reference as R

pytestmark = pytest.mark.gpu
TYPES = [np.float32, np.float64]


def ptr(buf, elements=0):
    return None if buf is None else buf.ptr + elements * buf.dtype.itemsize


def close(got, want, bound, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= bound + 1e-300)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3],
                           bound[bad][:3])


def strided(dev, a, pad, offset):
    """`a` (..., rows, cols) in a buffer whose rows are `pad` elements longer and start `offset` in, the
    rest holding NaN: (buffer, row stride)."""
    wide = np.full(a.shape[:-1] + (a.shape[-1] + pad,), np.nan, a.dtype)
    wide[..., offset:offset + a.shape[-1]] = a
    return dev.array(wide), a.shape[-1] + pad


# ---- rms_norm -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [
    (1, 1, 0), (3, 7, 0), (5, 64, 0), (4, 256, 4), (9, 1000, 3), (2, 1024, 0), (7, 1537, 0), (3, 2048, 8), (2, 4100, 0),
    (2, 8192, 0), (3, 8193, 1), (2, 40000, 0), (1, 70001, 0), (1000, 96, 0),
])
@pytest.mark.parametrize("form", ["plain", "residual", "in_place", "no_weight"])
def test_rms_norm(dev, dtype, rows, cols, pad, form):
    rng = np.random.default_rng(rows * 7 + cols)
    x = rng.standard_normal((rows, cols)).astype(dtype)
    res = None if form == "plain" else (3 * rng.standard_normal((rows, cols))).astype(dtype)
    w = None if form == "no_weight" else (1 + 0.1 * rng.standard_normal(cols)).astype(dtype)
    y, r, ey, er = R.rms_norm(x, res, w, 1e-6, R.half_step(dtype))
    dx, xs = strided(dev, x, pad, pad)
    dres = None if res is None else dev.array(res)
    dout = None if res is None else dres if form == "in_place" else dev.array(np.full_like(x, 77))
    dw = None if w is None else dev.array(w)
    dy = dev.array(np.full((rows + 1, cols + pad), 55, dtype))
    a = L.RmsNorm(H.DT[np.dtype(dtype)], rows, cols, ptr(dx, pad), xs, ptr(dres), cols, ptr(dout), cols, ptr(dw), 1e-6,
                  dy.ptr, cols + pad)
    L.check(L.lib.cnh_rms_norm(C.byref(a), None))
    got = dy.get()
    close(got[:rows, :cols], y, ey, "y")
    assert (got[rows] == 55).all() and (got[:rows, cols:] == 55).all()
    if res is not None:
        close(dout.get(), r, er, "residual_out")
    dev.free_all()


def test_rms_norm_of_nothing_and_of_what_is_no_number(dev):
    x = np.zeros((3, 40), np.float32)
    x[1] = np.inf
    x[2, 5] = np.nan
    dx, dy = dev.array(x), dev.array(np.full_like(x, 3))
    L.check(L.lib.cnh_rms_norm(C.byref(L.RmsNorm(L.F32, 3, 40, dx.ptr, 40, None, 0, None, 0, None, 1e-6, dy.ptr, 40)), None))
    got = dy.get()
    assert (got[0] == 0).all()               # a row of zeros stays one: eps keeps the root away from zero
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all()
    dev.free_all()


# ---- short_convolution ----------------------------------------------------------------------------


def conv_call(dev, dtype, x, w, bias, state, lengths, silu, in_place=False, time_major=False, pad=0):
    B, n, D = x.shape
    K = w.shape[0]
    lay = x.transpose(1, 0, 2) if time_major else x
    dx, xs = strided(dev, np.ascontiguousarray(lay), pad, 0)
    bs, ts = (xs, B * xs) if time_major else (n * xs, xs)
    dw, db = dev.array(w), None if bias is None else dev.array(bias)
    din = None if state is None else dev.array(state)
    dout = din if in_place else dev.array(np.full((B, max(K - 1, 1), D), 77, dtype))
    dl = None if lengths is None else dev.array(np.asarray(lengths, np.int32))
    dy = dev.array(np.full((B * n + 1, D), 55, dtype))
    ybs, yts = (D, B * D) if time_major else (n * D, D)
    a = L.ShortConvolution(H.DT[np.dtype(dtype)], int(silu), K, B, n, D, dx.ptr, bs, ts, dw.ptr, ptr(db), ptr(din),
                           dout.ptr, ptr(dl), dy.ptr, ybs, yts)
    L.check(L.lib.cnh_short_convolution(C.byref(a), None))
    got = dy.get()
    assert (got[B * n] == 55).all()
    y = got[:B * n].reshape((n, B, D)).transpose(1, 0, 2) if time_major else got[:B * n].reshape(B, n, D)
    return y, dout.get().reshape(B, -1, D)[:, :K - 1]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,n,D,K", [
    (1, 1, 1, 4), (2, 1, 64, 4), (3, 1, 4097, 2), (1, 2, 8, 8), (2, 7, 63, 4), (4, 8, 256, 3), (2, 9, 1100, 4),
    (3, 100, 129, 1), (1, 333, 36, 5), (2, 65, 1024, 4), (70, 3, 5, 6), (1, 40, 512, 7),
])
@pytest.mark.parametrize("form", ["bare", "full", "ragged", "in_place", "time_major"])
def test_short_convolution(dev, dtype, B, n, D, K, form):
    rng = np.random.default_rng(B * 1000 + n * 10 + D)
    x = rng.standard_normal((B, n, D)).astype(dtype)
    w = (0.5 * rng.standard_normal((K, D))).astype(dtype)
    bias = None if form == "bare" else (0.1 * rng.standard_normal(D)).astype(dtype)
    state = None if form == "bare" or K == 1 else rng.standard_normal((B, K - 1, D)).astype(dtype)
    lengths = None
    if form in ("ragged", "in_place"):
        lengths = rng.integers(0, n + 1, B)
        lengths[0] = -3 if form == "ragged" else n + 5     # held to 0 and to n
    silu = form != "ragged"
    y, after, bound = R.short_convolution(x, w, bias, state, lengths, silu, R.half_step(dtype))
    if lengths is not None:                                # what is behind a sequence must not matter
        for b in range(B):
            x[b, min(max(int(lengths[b]), 0), n):] = np.nan
    got, out = conv_call(dev, dtype, x, w, bias, state, lengths, silu, in_place=form == "in_place" and K > 1,
                         time_major=form == "time_major", pad=4 if form == "full" else 0)
    close(got, y, bound, "y")
    assert np.array_equal(out.astype(np.float64), after)
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
def test_convolution_of_a_cut_prompt_is_that_of_the_whole(dev, dtype):
    """A prompt in pieces of 0, 1, 2, 9 and 20 tokens, the state carried along: the same bits."""
    rng = np.random.default_rng(5)
    B, D, K = 2, 260, 4
    x = rng.standard_normal((B, 32, D)).astype(dtype)
    w, bias = rng.standard_normal((K, D)).astype(dtype), rng.standard_normal(D).astype(dtype)
    state = rng.standard_normal((B, K - 1, D)).astype(dtype)
    whole, last = conv_call(dev, dtype, x, w, bias, state, None, True)
    at, parts = 0, []
    for n in (1, 2, 9, 20):
        y, state = conv_call(dev, dtype, x[:, at:at + n], w, bias, np.ascontiguousarray(state), None, True)
        parts.append(y)
        at += n
    assert np.array_equal(np.concatenate(parts, axis=1), whole) and np.array_equal(state, last)
    # no token at all: the state passes through
    din, dout, dw = dev.array(state), dev.array(np.zeros_like(state)), dev.array(w)
    a = L.ShortConvolution(H.DT[np.dtype(dtype)], 0, K, B, 0, D, None, 0, 0, dw.ptr, None, din.ptr, dout.ptr, None, None,
                           0, 0)
    L.check(L.lib.cnh_short_convolution(C.byref(a), None))
    assert np.array_equal(dout.get(), state)
    dev.free_all()


# ---- state_scan -----------------------------------------------------------------------------------


def scan_inputs(dtype, B, n, D, N, seed):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s).astype(dtype)  # noqa: E731
    return dict(x=f(B, n, D), delta=(0.5 * f(B, n, D)).astype(dtype), z=f(B, n, D),
                A=(-np.arange(1, N + 1) * np.exp(0.1 * f(D, N))).astype(dtype), Bm=f(B, n, N), Cm=f(B, n, N),
                skip=f(D), delta_bias=rng.uniform(-6.9, -2.3, D).astype(dtype), state=f(B, D, N))


def scan_call(dev, dtype, q, lengths, softplus, in_place=False, time_major=False, pad=0):
    B, n, D = q["x"].shape
    N = q["A"].shape[1]

    def rows(a):
        if a is None:
            return None, 0, 0
        lay = np.ascontiguousarray(a.transpose(1, 0, 2) if time_major else a)
        buf, st = strided(dev, lay, pad, 0)
        return (buf.ptr, st, B * st) if time_major else (buf.ptr, n * st, st)
    opt = lambda k: None if q[k] is None else dev.array(q[k])  # noqa: E731
    dA, skip, db, din = dev.array(q["A"]), opt("skip"), opt("delta_bias"), opt("state")
    dout = din if in_place else dev.array(np.full((B, D, N), 77, dtype))
    dl = None if lengths is None else dev.array(np.asarray(lengths, np.int32))
    dy = dev.array(np.full((B * n + 1, D), 55, dtype))
    ybs, yts = (D, B * D) if time_major else (n * D, D)
    a = L.StateScan(H.DT[np.dtype(dtype)], int(softplus), B, n, D, N, *rows(q["x"]), *rows(q["delta"]), *rows(q["z"]),
                    dA.ptr, *rows(q["Bm"]), *rows(q["Cm"]), ptr(skip), ptr(db), ptr(din), dout.ptr, ptr(dl), dy.ptr, ybs,
                    yts, None, 0)
    need = L.check(L.lib.cnh_state_scan_workspace(C.byref(a)))
    if need:
        # what it holds at the start must not matter; the bytes behind it stay
        ws = dev.array(np.full(need // 4 + 64, np.nan, np.float32))
        a.workspace, a.workspace_bytes = ws.ptr, need
    L.check(L.lib.cnh_state_scan(C.byref(a), None))
    if need:
        assert np.isnan(ws.get()[need // 4:]).all()
    got = dy.get()
    assert (got[B * n] == 55).all()
    y = got[:B * n].reshape((n, B, D)).transpose(1, 0, 2) if time_major else got[:B * n].reshape(B, n, D)
    return y, dout.get(), need


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,n,D,N", [
    (1, 1, 1, 1), (2, 1, 64, 16), (3, 1, 129, 13), (2, 1, 70, 64), (1, 1, 33, 100), (2, 5, 64, 4), (1, 17, 65, 16),
    (2, 16, 300, 8), (1, 64, 64, 16), (1, 100, 130, 13), (2, 70, 40, 32), (1, 33, 20, 64), (1, 40, 9, 200),
    (1, 300, 96, 16), (3, 129, 256, 16), (1, 35, 8, 256), (2, 90, 31, 5),
])
@pytest.mark.parametrize("form", ["bare", "full", "ragged", "in_place", "time_major"])
def test_state_scan(dev, dtype, B, n, D, N, form):
    q = scan_inputs(dtype, B, n, D, N, B * 1000 + n * 10 + D + N)
    softplus, lengths = True, None
    if form == "bare":
        q.update(z=None, skip=None, delta_bias=None, state=None, delta=np.abs(q["delta"]) * dtype(0.1))
        softplus = False
    if form in ("ragged", "in_place"):
        lengths = np.random.default_rng(n).integers(0, n + 1, B)
        lengths[0] = -3 if form == "ragged" else n + 5
    y, h, ey, eh = R.state_scan(**q, lengths=lengths, softplus=softplus, u=R.half_step(dtype), piece=64)
    if lengths is not None:
        for b in range(B):
            for k in ("x", "delta", "z", "Bm", "Cm"):
                q[k][b, min(max(int(lengths[b]), 0), n):] = np.nan
    got, out, _ = scan_call(dev, dtype, q, lengths, softplus, in_place=form == "in_place",
                            time_major=form == "time_major", pad={"full": 4, "ragged": 3}.get(form, 0))
    close(got, y, ey, "y")
    close(out, h, eh, "state")
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_in_pieces_token_by_token_and_with_large_steps(dev, dtype):
    """A prompt that is cut along its tokens inside the call, the same prompt as a first part and single
    tokens, and steps so large that a state forgets at once (decays that underflow)."""
    B, n, D, N = 1, 700, 64, 16
    q = scan_inputs(dtype, B, n, D, N, 77)
    q["delta"][:, 100:110] = 30
    q["delta"][:, 300] = 200
    u = R.half_step(dtype)
    y, h, ey, eh = R.state_scan(**q, lengths=None, softplus=True, u=u, piece=64)
    got, out, need = scan_call(dev, dtype, q, None, True)
    assert need > 0
    close(got, y, ey, "y")
    close(out, h, eh, "state")
    part = {k: v[:, :690] if k in ("x", "delta", "z", "Bm", "Cm") else v for k, v in q.items()}
    first, state, _ = scan_call(dev, dtype, part, None, True)
    close(first, y[:, :690], ey[:, :690], "y of the first part")
    for t in range(690, 700):
        tok = {k: v[:, t:t + 1] if k in ("x", "delta", "z", "Bm", "Cm") else v for k, v in q.items()}
        tok["state"] = state
        yt, state, _ = scan_call(dev, dtype, tok, None, True, in_place=True)
        close(yt[:, 0], y[:, t], ey[:, t], f"token {t}")
    close(state, h, eh, "state after the tokens")
    dev.free_all()


def test_scan_without_tokens_keeps_the_state(dev):
    state = np.random.default_rng(1).standard_normal((2, 40, 16)).astype(np.float32)
    A = dev.array(-np.ones((40, 16), np.float32))
    din, dout = dev.array(state), dev.array(np.zeros_like(state))
    a = L.StateScan(L.F32, 1, 2, 0, 40, 16)
    a.A, a.state_in, a.state_out = A.ptr, din.ptr, dout.ptr
    L.check(L.lib.cnh_state_scan(C.byref(a), None))
    assert np.array_equal(dout.get(), state)
    dev.free_all()


# ---- sample_tokens --------------------------------------------------------------------------------


def sample_call(dev, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, pad=0):
    Rn, V = logits.shape
    dl, st = strided(dev, logits, pad, 0)
    du, out = dev.array(np.asarray(u, np.float64)), dev.array(np.full(Rn + 1, 55, np.int32))
    a = L.SampleTokens(H.DT[logits.dtype], 0, Rn, V, dl.ptr, st, du.ptr, 1.0, 1.0, 0.0)
    for name, v, t in (("temperature", temperature, np.float64), ("top_k", top_k, np.int32), ("top_p", top_p, np.float64),
                       ("min_p", min_p, np.float64)):
        if np.ndim(v):
            setattr(a, name + "s", dev.array(np.asarray(v, t)).ptr)
        else:
            setattr(a, name, v)
    a.out = out.ptr
    need = L.check(L.lib.cnh_sample_tokens_workspace(C.byref(a)))
    if need:
        ws = dev.array(np.full(need, 0xA5, np.uint8))
        a.workspace, a.workspace_bytes = ws.ptr, need
    L.check(L.lib.cnh_sample_tokens(C.byref(a), None))
    got = out.get()
    assert got[Rn] == 55
    return got[:Rn]


def check_rows(got, logits, u, temperature, top_k, top_p, min_p):
    at = lambda v, r: v[r] if np.ndim(v) else v  # noqa: E731
    for r in range(len(u)):
        want, near = R.sample_tokens(logits[r], u[r], at(temperature, r), at(top_k, r), at(top_p, r), at(min_p, r))
        # Masses are multiples of 2^-45 (relative to a sum of at least 1): the running sums of V words are
        # off by V 2^-46 at most; nearer than that to a border the draw may go either way.
        if near > logits.shape[1] * 2.0 ** -45:
            assert got[r] == want, (r, got[r], want, near)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,pad", [(1, 0), (2, 0), (5, 3), (64, 0), (1000, 0), (1023, 1), (5003, 0), (50021, 0), (131072, 0)])
@pytest.mark.parametrize("temperature,top_k,top_p,min_p", [
    (1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 50, 1.0, 0.0), (1.3, 50, 0.9, 0.01),
    (1.0, 1, 1.0, 0.0), (0.0, 50, 0.9, 0.0), (1.0, 2000, 0.95, 0.0), (2.0, 40000, 0.99, 0.001), (1.0, 3, 0.0, 0.0),
    (30.0, 0, 0.7, 0.0), (30.0, 30000, 0.9, 0.1), (0.01, 0, 0.9, 1.0),
])
def test_sample_tokens(dev, dtype, V, pad, temperature, top_k, top_p, min_p):
    rng = np.random.default_rng(V + top_k)
    logits = (2.5 * rng.standard_normal((6, V))).astype(dtype)
    logits[1:3][rng.random((2, V)) < 0.3] = -np.inf
    u = rng.random(6)
    u[0], u[5] = 0.0, 1 - 2.0 ** -53
    got = sample_call(dev, logits, u, temperature, top_k, top_p, min_p, pad)
    check_rows(got, logits, u, temperature, top_k, top_p, min_p)
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (7, 1.0, 0.0), (700, 0.5, 0.0), (5000, 0.9, 0.0), (0, 0.3, 0.5)])
def test_sample_ties_and_crowds(dev, dtype, top_k, top_p, min_p):
    """Rows of one value, of few values and of values so close together that no histogram of depths
    separates them: ties go to the lowest index, crowded bins are split by the values' bits."""
    rng = np.random.default_rng(3)
    V = 20000
    rows = [np.zeros(V), rng.integers(0, 3, V), 1 + 1e-4 * rng.random(V), np.where(rng.random(V) < 0.5, 0.0, -0.0),
            np.repeat([5.0, 4.999, -3.0, 5.0], V // 4), 1e-3 * rng.integers(0, 5000, V) / 5000 + 4]
    logits = np.stack(rows).astype(dtype)
    u = rng.random(len(rows))
    got = sample_call(dev, logits, u, 1.0, top_k, top_p, min_p)
    check_rows(got, logits, u, 1.0, top_k, top_p, min_p)
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_masks_and_what_is_no_number(dev, dtype):
    V = 300
    low = np.finfo(dtype).min
    logits = np.zeros((10, V), dtype)
    logits[0] = -np.inf                       # nothing left
    logits[1] = np.nan
    logits[2] = -np.inf
    logits[2, 17] = -5                        # one left
    logits[3] = low                           # all masked by the lowest value: all alike
    logits[4] = low
    logits[4, 200] = 0                        # one that is not
    logits[5, 3:7] = np.inf                   # infinities share the mass
    logits[6, ::2] = np.nan
    logits[6, 1::2] = np.linspace(-1, 1, 150)
    logits[7, :] = -np.inf
    logits[7, 100:] = np.nan
    logits[8, 250] = np.nan
    logits[9] = np.linspace(-1e30, 1e30, V)   # the next one is out of reach of any temperature near 1
    u = np.array([0.5, 0.5, 0.9, 0.5, 0.999, 0.6, 0.3, 0.5, 0.5, 0.999999])
    got = sample_call(dev, logits, u)
    want = [R.sample_tokens(logits[r], u[r], 1.0, 0, 1.0, 0.0)[0] for r in range(10)]
    assert want[0] == want[1] == want[7] == -1 and want[2] == 17 and want[4] == 200 and want[9] == V - 1
    assert want[3] == 150 and want[5] == 5
    assert got.tolist() == want
    # greedy rows of the same
    got = sample_call(dev, logits, u, temperature=0.0)
    assert got.tolist() == [R.sample_tokens(logits[r], u[r], 0.0, 0, 1.0, 0.0)[0] for r in range(10)]
    dev.free_all()


def test_sample_settings_per_row(dev):
    rng = np.random.default_rng(8)
    Rn, V = 40, 7001
    logits = (3 * rng.standard_normal((Rn, V))).astype(np.float32)
    u = rng.random(Rn)
    t, k = rng.uniform(0.3, 2, Rn), rng.integers(0, 3000, Rn)
    p, m = rng.uniform(0.5, 1.1, Rn), rng.uniform(0, 0.1, Rn)
    t[0], t[1], k[2], p[3], m[4], m[5] = 0.0, -1.0, -4, 2.0, 0.0, 7.0      # out of range: held to it
    got = sample_call(dev, logits, u, t, k, p, m)
    check_rows(got, logits, u, t, k, p, m)
    assert got[0] == np.argmax(logits[0]) and got[1] == np.argmax(logits[1]) and got[5] == np.argmax(logits[5])
    # random numbers outside [0, 1) are held to it as well
    u[:4] = [-1.0, np.nan, 1.0, 5.0]
    got = sample_call(dev, logits, u, 1.0, 3)
    order = np.argsort(-logits[:4].astype(np.float64), axis=1, kind="stable")
    assert got[:4].tolist() == [order[0, 0], order[1, 0], order[2, 2], order[3, 2]]
    dev.free_all()


def test_sample_follows_the_weights(dev):
    """Evenly spread random numbers draw each word as often as its weight says."""
    rng = np.random.default_rng(4)
    V, n = 37, 4000
    one = rng.standard_normal(V).astype(np.float32)
    got = sample_call(dev, np.repeat(one[None], n, axis=0), (np.arange(n) + 0.5) / n)
    w = np.exp(one.astype(np.float64))
    # n evenly spaced numbers meet an interval of length l between n l - 1 and n l + 1 times
    assert (np.abs(np.bincount(got, minlength=V) - n * w / w.sum()) <= 1 + 1e-6).all()
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
def test_sample_few_long_rows(dev, dtype):
    """Rows long enough to be weighed in slices, all kinds of them in one call: the slices of rows that are
    not weighed, masked or infinite, and crowds that lie in several slices."""
    rng = np.random.default_rng(12)
    V = 40003
    x = (2 * rng.standard_normal((12, V))).astype(dtype)
    x[3] = -np.inf
    x[4, 5:V:7] = np.inf
    x[5] = np.finfo(dtype).min
    x[6] = 1.5
    x[7, : V // 2] = -np.inf                              # nothing in the first slices
    x[8] = np.nan
    x[9, 1:] = -np.inf                                    # a single word
    x[10] = rng.integers(0, 2, V)
    u = rng.random(12)
    t = np.array([1.0, 0.8, 0.0, 1, 1, 1, 1, 1.2, 1, 1, 0.9, 2.0])
    k = np.array([0, 3, 7, 0, 9000, 0, 30000, 0, 0, 0, 25000, 5000])
    p = np.array([0.9, 0.9, 1, 1, 0.4, 0.7, 0.6, 1.0, 1, 0.3, 0.99, 0.8])
    m = np.array([0, 0, 0, 0, 0.1, 0.5, 0, 0.01, 0, 0.2, 0, 0])
    got = sample_call(dev, x, u, t, k, p, m)
    check_rows(got, x, u, t, k, p, m)
    assert got[3] == got[8] == -1 and got[9] == 0 and got[4] % 7 == 5
    again = sample_call(dev, x, u, t, k, p, m)
    assert np.array_equal(got, again)
    one = np.concatenate([sample_call(dev, x[r:r + 1], u[r:r + 1], t[r], int(k[r]), p[r], m[r]) for r in range(12)])
    assert np.array_equal(got, one)                       # the same word however many rows and slices there are
    dev.free_all()
