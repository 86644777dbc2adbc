"""The sequence operators at the limits of what they document: states that grow, prompts in more pieces than one
round of the carry pass takes, infinite inputs, the precision of the functions they apply, crowds of equal words,
counts beyond 32 bits."""
import ctypes as C

import numpy as np
import pytest

import charmnumeric_amd as cnp
from charmnumeric_amd import _lib as L
from tests import helpers as H
from tests import sequence_reference as R
from tests.test_gpu_sequence import close, conv_call, sample_call, scan_call, scan_inputs

pytestmark = pytest.mark.gpu
TYPES = [np.float32, np.float64]
TOKENS = ("x", "delta", "z", "Bm", "Cm")


# ---- the carry pass of a cut scan -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start", ["zero", "tiny"])
def test_cut_scan_of_growing_states(dev, dtype, start):
    """States that grow by more than the type's range over several pieces, from nothing and from a number as
    small as the type has: the state itself stays in range. Cut, and in parts that are not cut."""
    B, n, D, N = 1, 700, 64, 16
    q = scan_inputs(dtype, B, n, D, N, 21)
    step = 0.7 if dtype == np.float32 else 6.0                # e^95, e^816 over eight pieces of 17 tokens
    q.update(z=None, skip=None, delta_bias=None)
    q["delta"][:] = step
    q["A"][:, ::2], q["A"][:, 1::2] = 1.0, -0.5
    q["x"][:, :640] = 0
    if start == "zero":
        q["state"] = None
    else:
        q["state"][:] = 1e-36 if dtype == np.float32 else 1e-300
        q["delta"][:, 170:] = 0                               # 1e-36 e^119 = 5e15, 1e-300 e^1020 = 1e143
    y, h, ey, eh = R.state_scan(**q, lengths=None, softplus=False, u=R.half_step(dtype), piece=64)
    assert np.isfinite(y).all() and np.abs(h).max() > 1e10 and (start == "zero" or np.abs(y[0, 600]).min() > 1e10)
    got, out, need = scan_call(dev, dtype, q, None, False)
    assert need > 0
    close(got, y, ey, "y")
    # The states that shrink do so by 0.705 or less a token (e^-0.35) until they are below the type's smallest
    # normal number, where a product loses that number at most: 1 / (1 - 0.705) < 4 of it in all.
    close(out, h, eh + 4 * float(np.finfo(dtype).tiny), "state")
    state = q["state"]
    for at in range(0, n, 90):
        part = {k: v[:, at:at + 90] if k in TOKENS and v is not None else v for k, v in q.items()}
        part["state"] = state
        got, state, need = scan_call(dev, dtype, part, None, False)
        assert need == 0
        close(got, y[:, at:at + 90], ey[:, at:at + 90], f"y from token {at}")
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,lengths", [(1100, None), (2100, None), (1100, [137]), (2100, [1700])])
def test_scan_in_more_pieces_than_a_round(dev, dtype, n, lengths):
    """65 and 124 pieces, where one round of the carry pass takes 64: what a round leaves starts the next, also
    when the sequence ends in the first round. The state is updated in place."""
    B, D, N = 1, 64, 16
    q = scan_inputs(dtype, B, n, D, N, n)
    q["A"] = (q["A"] / 40).astype(dtype)                      # what the first round leaves is still there in the last
    y, h, ey, eh = R.state_scan(**q, lengths=lengths, softplus=True, u=R.half_step(dtype), piece=64)
    got, out, need = scan_call(dev, dtype, q, lengths, True, in_place=True)
    assert need // (np.dtype(dtype).itemsize * (N + 1) * D) == (65 if n == 1100 else 124)
    close(got, y, ey, "y")
    close(out, h, eh, "state")
    dev.free_all()


# ---- infinite inputs ------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 40, 700])
@pytest.mark.parametrize("N", [1, 3, 5, 13, 16, 29, 50, 100, 130])
@pytest.mark.parametrize("skip", [True, False])
def test_scan_of_infinite_inputs(dev, dtype, n, N, skip):
    """An infinite x makes its channel's states and results infinite from there on, and no other's, also where
    the rows of states are not full and where the call has no skip."""
    D, bad, u = 70, n // 2, R.half_step(dtype)
    q = scan_inputs(dtype, 1, n, D, N, n + N)
    q["delta"][:] = 0.05
    q["A"][:] = -np.arange(1, N + 1)
    for k in ("Bm", "Cm"):
        q[k] = (np.abs(q[k]) + 0.1).astype(dtype)
    q.update(z=None, skip=np.abs(q["skip"]) + dtype(0.1) if skip else None, delta_bias=None)
    y, h, ey, eh = R.state_scan(**q, lengths=None, softplus=False, u=u, piece=64)
    q["x"][0, bad, 5], q["x"][0, bad, 66] = np.inf, -np.inf
    got, out, _ = scan_call(dev, dtype, q, None, False)
    for d, v in ((5, np.inf), (66, -np.inf)):
        assert (got[0, bad:, d] == v).all() and (out[0, d] == v).all(), (got[0, bad:, d], out[0, d])
        got[0, bad:, d], out[0, d] = y[0, bad:, d], h[0, d]
    close(got, y, ey, "y")
    close(out, h, eh, "state")
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [5, 12, 16, 20])
@pytest.mark.parametrize("skip", [True, False])
def test_scan_of_infinite_inputs_in_many_sequences(dev, dtype, N, skip):
    """The same in batches that fill the device, where a lane has all states of a channel."""
    B, n, D, bad, u = 1100, 33, 64, 11, R.half_step(dtype)
    q = scan_inputs(dtype, 1, n, D, N, N)
    q["delta"][:] = 0.05
    q["A"][:] = -np.arange(1, N + 1)
    for k in ("Bm", "Cm"):
        q[k] = (np.abs(q[k]) + 0.1).astype(dtype)
    q.update(z=None, skip=np.abs(q["skip"]) + dtype(0.1) if skip else None, delta_bias=None)
    y, h, ey, eh = R.state_scan(**q, lengths=None, softplus=False, u=u)
    q["x"][0, bad, 5] = np.inf
    one, rep = {k: dev.array(v) for k, v in q.items() if v is not None}, dev.array(np.repeat(q["state"], B, axis=0))
    dy = dev.array(np.full((B, n, D), 7, dtype))
    a = L.StateScan(H.DT[np.dtype(dtype)], 0, B, n, D, N, one["x"].ptr, 0, D, one["delta"].ptr, 0, D, None, 0, 0, one["A"].ptr,
                    one["Bm"].ptr, 0, N, one["Cm"].ptr, 0, N, one["skip"].ptr if skip else None, None, rep.ptr, rep.ptr, None, dy.ptr, n * D, D)
    assert L.lib.cnh_state_scan_workspace(C.byref(a)) == 0
    L.check(L.lib.cnh_state_scan(C.byref(a), None))
    got, hs = dy.get(), rep.get()
    assert (got == got[:1]).all() and (hs == hs[:1]).all()
    assert (got[0, bad:, 5] == np.inf).all() and (hs[0, 5] == np.inf).all()
    got, hs = got[:1].copy(), hs[:1].copy()
    got[0, bad:, 5], hs[0, 5] = y[0, bad:, 5], h[0, 5]
    close(got, y, ey, "y")
    close(hs, h, eh, "state")
    dev.free_all()


# ---- the functions' own precision -----------------------------------------------------------------


def spread(dtype, far, seed, n=40000):
    """Numbers of every size up to `far`, of both signs."""
    rng = np.random.default_rng(seed)
    v = np.concatenate([rng.uniform(-far, far, n), rng.uniform(-20, 20, n), np.exp(rng.uniform(-9, 0, n)) * rng.choice([-1, 1], n)])
    return v.astype(dtype)


def within(got, want, half_steps, v, dtype, what):
    """got is off from want by so many half steps of the type at most (relative to want)."""
    e = np.abs((got.astype(np.longdouble) - want) / want) / R.half_step(dtype)
    over = ~(e <= half_steps)
    assert not over.any(), (what, int(over.sum()), float(e[over].max()), v[over][:4], e[over][:4].astype(float))


@pytest.mark.parametrize("dtype", TYPES)
def test_precision_of_the_activation(dev, dtype):
    """v sigmoid(v), through a convolution of one tap. e^-v to within 2.2 half steps in 64 bits (its remainder
    0.35, its polynomial 0.25 and 1.5), 1 + e^-v, quotient and product 1 each. In 32 bits the hardware's exponential
    (an ulp, 2 half steps; log 2 in 24 bits 0.046 |v|), what its argument's rounding left, 1 + e^-v and the product 1
    each, the reciprocal 2."""
    v = spread(dtype, 80 if dtype == np.float32 else 690, 1)
    v = v[v != 0]
    got, _ = conv_call(dev, dtype, v.reshape(1, 1, -1), np.ones((1, v.size), dtype), None, None, None, True)
    x = v.astype(np.longdouble)
    within(got.reshape(-1), x / (1 + np.exp(-x)), 7.5 + 0.05 * np.abs(v) if dtype == np.float32 else 6.0, v, dtype, "silu")
    ends = np.array([0.0, -0.0, np.inf, -1e30, 1e30, np.nan, -1000], dtype)
    got, _ = conv_call(dev, dtype, ends.reshape(1, 1, -1), np.ones((1, ends.size), dtype), None, None, None, True)
    assert np.array_equal(got.reshape(-1), np.array([0, 0, np.inf, 0, 1e30, np.nan, 0], dtype), equal_nan=True)
    dev.free_all()


def one_token(dtype, D, **kw):
    """A scan of one token and one state per channel: y = exp(s A) h + s."""
    q = dict(x=np.ones((1, 1, D), dtype), delta=np.zeros((1, 1, D), dtype), z=None, A=np.zeros((D, 1), dtype),
             Bm=np.ones((1, 1, 1), dtype), Cm=np.ones((1, 1, 1), dtype), skip=None, delta_bias=None, state=None)
    q.update(kw)
    return q


@pytest.mark.parametrize("dtype", TYPES)
def test_precision_of_the_step(dev, dtype):
    """log(1 + e^v). 64 bits: e^-|v| 2.2 half steps, denominator, quotient and its last product 1 each, the sum 1.
    32 bits: exponential 2 (and 0.046 |v|), logarithm 2 and a product, reciprocal 2 and two products, and what of the
    rounding of 1 + e^v does not cancel, 1."""
    v = spread(dtype, 80 if dtype == np.float32 else 690, 2)
    y, _, _ = scan_call(dev, dtype, one_token(dtype, v.size, delta=v.reshape(1, 1, -1)), None, True)
    x = v.astype(np.longdouble)
    within(y.reshape(-1), np.log1p(np.exp(-np.abs(x))) + np.maximum(x, 0), 10 + 0.05 * np.abs(v) if dtype == np.float32 else 6.2, v,
           dtype, "softplus")
    ends = np.array([-np.inf, np.inf, np.nan, -1e30, 1e30, 0], dtype)
    y, _, _ = scan_call(dev, dtype, one_token(dtype, ends.size, delta=ends.reshape(1, 1, -1), x=np.ones((1, 1, ends.size), dtype)),
                        None, True)
    assert np.array_equal(y.reshape(-1)[[0, 3, 4]], np.array([0, 0, 1e30], dtype)) and np.isnan(y.reshape(-1)[2])
    assert abs(y.reshape(-1)[5] - np.log(2)) < 4 * R.half_step(dtype)
    dev.free_all()


def test_precision_of_the_decay(dev):
    """exp(s A) in 64 bits: one rounding of A log2(e) (and 0.13 of its constant's), each |s A| half steps, and the
    exponential's 2.2. What e^(s A) of a single state loses by rounding s A alone is |s A|."""
    rng = np.random.default_rng(3)
    n = 60000
    s = np.exp(rng.uniform(-8, 3, n))
    A = -rng.uniform(0, 100, n) / s
    A[:n // 8] *= -1
    zero = np.zeros((1, 1, n))
    y, _, _ = scan_call(dev, np.float64, one_token(np.float64, n, x=zero, delta=s.reshape(1, 1, -1), A=A.reshape(-1, 1),
                                                   state=np.ones((1, n, 1))), None, False)
    t = s.astype(np.longdouble) * A.astype(np.longdouble)
    within(y.reshape(-1), np.exp(t), 1.2 * np.abs(s * A) + 3.2, s * A, np.float64, "decay")
    # far arguments on both sides, and none
    s = np.array([1e21, 1e21, 1.0, 0.0, 3.0, 1e10, 1e10])
    A = np.array([-1e21, 1e21, -1e5, -np.inf, -np.inf, 1e10, -1e10])
    y, _, _ = scan_call(dev, np.float64, one_token(np.float64, 7, x=np.zeros((1, 1, 7)), delta=s.reshape(1, 1, -1),
                                                   A=A.reshape(-1, 1), state=np.ones((1, 7, 1))), None, False)
    assert y.reshape(-1).tolist() == [0, np.inf, 0, 1, 0, np.inf, 0]
    dev.free_all()


# ---- the norm's eps -------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,eps", [(np.float32, 1e-50), (np.float32, 1e-45), (np.float32, 1e-39), (np.float64, 5e-324)])
def test_norm_of_zeros_with_an_eps_below_the_type(dev, dtype, eps):
    """An eps that is not zero keeps a row of zeros one, however small it is."""
    for cols in (40, 41, 9000):
        x = np.zeros((2, cols), dtype)
        x[1] = 1
        dx, dy = dev.array(x), dev.array(np.full_like(x, 3))
        a = L.RmsNorm(H.DT[np.dtype(dtype)], 2, cols, dx.ptr, cols, None, 0, None, 0, None, eps, dy.ptr, cols)
        L.check(L.lib.cnh_rms_norm(C.byref(a), None))
        got = dy.get()
        assert (got[0] == 0).all() and np.abs(got[1] - 1).max() <= 8 * R.half_step(dtype)
    dev.free_all()


# ---- crowds of equal words ------------------------------------------------------------------------


def crowds(dtype):
    rng = np.random.default_rng(3)
    V = 20000
    rows = [np.zeros(V), rng.integers(0, 3, V), 1 + 1e-4 * rng.random(V), np.where(rng.random(V) < 0.5, 0.0, -0.0),
            np.repeat([5.0, 4.999, -3.0, 5.0], V // 4), 1e-3 * rng.integers(0, 5000, V) / 5000 + 4]
    return np.stack(rows).astype(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top_k,top_p,min_p", [(700, 0.50031, 0.0), (5000, 0.90017, 0.0), (0, 0.30013, 0.5), (12001, 0.77777, 0.2),
                                               (300, 0.50113, 0.0), (19999, 0.99987, 0.0)])
def test_sample_crowds_cut_between_words(dev, dtype, top_k, top_p, min_p):
    """Cuts that fall clearly between two words of a crowd, and draws that do: every row is checked."""
    logits = crowds(dtype)
    u = np.array([0.31417, 0.62713, 0.50123, 0.87117, 0.99991, 0.01237])
    want = [R.sample_tokens(logits[r], u[r], 1.0, top_k, top_p, min_p) for r in range(len(u))]
    assert min(near for _, near in want) > logits.shape[1] * 2.0 ** -45
    got = sample_call(dev, logits, u, 1.0, top_k, top_p, min_p)
    assert got.tolist() == [w for w, _ in want]
    for r in range(len(u)):                                   # few rows are weighed in slices, one by one too
        assert sample_call(dev, logits[r:r + 1], u[r:r + 1], 1.0, top_k, top_p, min_p)[0] == got[r]
    dev.free_all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top_k,top_p", [(700, 0.5), (5000, 0.9), (0, 0.3), (300, 0.25)])
def test_sample_crowds_cut_at_a_word(dev, dtype, top_k, top_p):
    """Rows of one value where top_p of top_k is a whole number of words: the cut is at that word or, as
    the product rounds, the one after it, and the word drawn follows from the cut."""
    V = 20000
    u = np.array([0.0, 0.31417, 0.62713, 0.87117, 0.99991])
    logits = np.repeat(np.array([[0.0], [-7.5], [3.0], [np.finfo(dtype).min], [1.0]]), V, axis=1).astype(dtype)
    whole = round(top_p * (top_k or V))
    got = sample_call(dev, logits, u, 1.0, top_k, top_p)
    for r in range(len(u)):
        assert got[r] in {int(u[r] * whole), int(u[r] * (whole + 1))}, (r, got[r], whole)
    dev.free_all()


# ---- counts beyond 32 bits ------------------------------------------------------------------------


@pytest.fixture(params=["plain", "tiles", "pipeline"])
def itf(request):
    cnp.reset()
    it = cnp.CharmNumericInterface(device=0)
    it.connect(odf=64 if request.param == "tiles" else 4)
    if request.param == "tiles":
        it.set_min_tile(1, 2)
    if request.param == "pipeline":
        it.set_pipeline()
    yield it
    cnp.reset()
    it.close()


@pytest.mark.parametrize("where", ["host", "array", "slice"])
def test_counts_of_64_bits_are_held_to_their_range(itf, where):
    """lengths and top_k of 64-bit integers mean what they say: beyond the sequence all of it, negative none."""
    rng = np.random.default_rng(6)

    def given(values):
        v = np.array(values, np.int64)
        if where == "host":
            return v
        if where == "array":
            return cnp.array(v)
        return cnp.array(np.concatenate([[7], v, [9]]))[1:-1]

    x, w = rng.standard_normal((5, 9, 8)), rng.standard_normal((3, 8))
    lengths = [2 ** 32 + 3, -2 ** 40, 4, 2 ** 31, -2 ** 32 + 2]
    y, _, ey = R.short_convolution(x, w, None, None, [9, 0, 4, 9, 0], True, R.half_step(np.float64))
    got = cnp.short_convolution(cnp.array(x), cnp.array(w), lengths=given(lengths)).get(itf)
    close(got, y, ey, "convolution")
    q = scan_inputs(np.float64, 5, 9, 8, 4, 1)
    a = {k: cnp.array(v) for k, v in q.items()}
    y, h, ey, eh = R.state_scan(**q, lengths=[9, 0, 4, 9, 0], softplus=True, u=R.half_step(np.float64))
    got = cnp.state_scan(a["x"], a["delta"], a["A"], a["Bm"], a["Cm"], a["skip"], a["z"], a["delta_bias"], a["state"],
                         given(lengths))
    close(got.get(itf), y, ey, "scan")
    close(a["state"].get(itf), h, eh, "state")

    logits, u = 2 * rng.standard_normal((5, 300)), rng.random(5)
    ks = [2 ** 32 + 1, 2 ** 31 + 3, 5, -2 ** 32 + 1, 2 ** 33]
    got = cnp.random.sample_tokens(cnp.array(logits), u, 1.0, given(ks)).get(itf)
    want = [R.sample_tokens(logits[r], u[r], 1.0, k, 1.0, 0.0)[0] for r, k in enumerate([0, 0, 5, 0, 0])]
    assert got.tolist() == want
