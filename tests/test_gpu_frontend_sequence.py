"""The sequence operators through the frontend and the executor: the decode loop of a small recurrent
model, cut and uncut arrays, slices, the asynchronous executor."""
import numpy as np
import pytest

import charmnumeric_amd as cnp
from tests import sequence_reference as R
from tests.test_gpu_sequence import close, scan_inputs

pytestmark = pytest.mark.gpu

SETUPS = {"default": {}, "tiles": dict(min_tile=8), "tiles_apart": dict(min_tile=8, layout=False),
          "solver": dict(min_tile=8, layout=False, solver=True), "pipeline": dict(pipeline=True)}


@pytest.fixture(params=sorted(SETUPS))
def itf(request):
    cnp.reset()
    how = SETUPS[request.param]
    it = cnp.CharmNumericInterface(device=0)
    it.connect(odf=64 if "min_tile" in how else 4)
    if "min_tile" in how:
        for nd in (1, 2, 3):
            it.set_min_tile(nd, how["min_tile"])
    if "layout" in how:
        it.set_layout(how["layout"])
    if how.get("solver"):
        it.set_solver()
    if how.get("pipeline"):
        it.set_pipeline()
    yield it
    cnp.reset()
    it.close()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_each_operator_against_its_definition(itf, dtype):
    u = R.half_step(dtype)
    rng = np.random.default_rng(2)
    B, n, D, N = 3, 21, 40, 16
    q = scan_inputs(dtype, B, n, D, N, 6)
    lengths = [21, 0, 9]
    xz = rng.standard_normal((B, n, 2 * D)).astype(dtype)
    q["z"] = xz[:, :, D:]
    y, h, ey, eh = R.state_scan(**q, lengths=lengths, softplus=True, u=u, piece=64)
    a = {k: cnp.array(v) for k, v in q.items() if k != "z"}
    dxz = cnp.array(xz)
    got = cnp.state_scan(a["x"], a["delta"], a["A"], a["Bm"], a["Cm"], a["skip"], dxz[:, :, D:], a["delta_bias"],
                         a["state"], lengths)
    close(got.get(itf), y, ey, "scan")
    close(a["state"].get(itf), h, eh, "scan state")

    w, bias = rng.standard_normal((4, D)).astype(dtype), rng.standard_normal(D).astype(dtype)
    st = rng.standard_normal((B, 3, D)).astype(dtype)
    y, after, ey = R.short_convolution(xz[:, :, :D], w, bias, st, lengths, True, u)
    dst = cnp.array(st)
    got = cnp.short_convolution(dxz[:, :, :D], w, bias, dst, np.array(lengths))
    close(got.get(itf), y, ey, "convolution")
    assert np.array_equal(dst.get(itf), after.astype(dtype))

    res, g = rng.standard_normal((B, n, D)).astype(dtype), rng.standard_normal(D).astype(dtype)
    dres = cnp.array(res)
    y, r, ey, er = R.rms_norm(xz[:, :, 3:3 + D].reshape(-1, D), res.reshape(-1, D), g, 1e-5, u)
    got = cnp.rms_norm(dxz[:, :, 3:3 + D], g, dres, eps=1e-5)
    close(got.get(itf).reshape(-1, D), y, ey, "norm")
    close(dres.get(itf).reshape(-1, D), r, er, "residual")
    y, r, ey, er = R.rms_norm(xz[:, 4:, :].reshape(-1, 2 * D), None, None, 1e-6, u)
    close(cnp.rms_norm(dxz[:, 4:, :]).get(itf).reshape(-1, 2 * D), y, ey, "norm of a slice")
    y, r, ey, er = R.rms_norm(res[0, 0][None], None, None, 1e-6, u)
    close(cnp.rms_norm(cnp.array(res[0, 0])).get(itf)[None], y, ey, "norm of a vector")

    logits = (2 * rng.standard_normal((5, 333))).astype(dtype)
    un, ks = rng.random(5), np.array([0, 1, 5, 50, 400])
    got = cnp.random.sample_tokens(cnp.array(logits), un, 0.8, ks, 0.9, 0.01).get(itf)
    assert got.dtype == np.int32
    assert got.tolist() == [R.sample_tokens(logits[r], un[r], 0.8, ks[r], 0.9, 0.01)[0] for r in range(5)]
    one = cnp.random.sample_tokens(cnp.array(logits)[2:3, 10:300], un[:1], top_p=0.5).get(itf)
    assert one.tolist() == [R.sample_tokens(logits[2, 10:300], un[0], 1.0, 0, 0.5, 0.0)[0]]


class Model:
    """Two blocks of norm, convolution and scan between products, and a head: on Arrays."""

    def __init__(self, dtype, D=48, N=8, K=4, V=200, seed=11):
        rng = np.random.default_rng(seed)
        f = lambda *s: (rng.standard_normal(s) / np.sqrt(s[0])).astype(dtype)  # noqa: E731
        self.D, self.N, self.K, self.V, self.dtype = D, N, K, V, dtype
        self.embed = f(V, D) * dtype(7)
        self.head = f(D, V)
        self.blocks = []
        for _ in range(2):
            self.blocks.append(dict(
                g=(1 + 0.1 * f(D)).astype(dtype), w_in=f(D, 2 * D), conv=f(K, D), bias=f(D), w_x=f(D, D + 2 * N),
                A=(-np.arange(1, N + 1) * np.exp(0.1 * f(D, N))).astype(dtype), skip=f(D),
                db=rng.uniform(-4, -2, D).astype(dtype), w_out=f(D, D)))


def forward(m, p, x, state, B, n, norm, conv, scan, mat):
    """One pass of n tokens for each of B sequences: logits of every token, (B * n, V)."""
    res = None
    for blk, st in zip(p, state):
        h, res = norm(x, blk["g"], res)
        xz = mat(h, blk["w_in"])
        c = conv(xz, blk, st, B, n, m.D)
        par = mat(c, blk["w_x"])
        y = scan(c, par, xz, blk, st, B, n, m.D, m.N)
        x = mat(y, blk["w_out"])
    h, res = norm(x, None, res)
    return mat(h, p_head(p))


def p_head(p):
    return p[-1]["head"]


def test_decode_loop_of_a_model(itf):
    """A prompt, then tokens drawn one by one, in double precision: every logit against the same model
    in NumPy, every word against the draw from those logits, and the states carried along give what the whole
    sequence gives in one pass."""
    dtype, u = np.float64, R.half_step(np.float64)
    m = Model(dtype)
    B, n, steps = 3, 11, 6
    rng = np.random.default_rng(1)
    words = rng.integers(0, m.V, (B, n))
    us = rng.random((steps, B))

    def np_norm(x, g, res):
        y, r, _, _ = R.rms_norm(x, res, g, 1e-6, u)
        return y, r

    def np_conv(xz, blk, st, B, n, D):
        y, st["conv"], _ = R.short_convolution(xz[:, :D].reshape(B, n, D), blk["conv"], blk["bias"], st["conv"], None, True, u)
        return y.reshape(B * n, D)

    def np_scan(c, par, xz, blk, st, B, n, D, N):
        y, st["h"], _, _ = R.state_scan(c.reshape(B, n, D), par[:, :D].reshape(B, n, D), xz[:, D:].reshape(B, n, D),
                                        blk["A"], par[:, D:D + N].reshape(B, n, N), par[:, D + N:].reshape(B, n, N),
                                        blk["skip"], blk["db"], st["h"], None, True, u)
        return y.reshape(B * n, D)

    def fresh(make):
        return [dict(conv=make((B, m.K - 1, m.D)), h=make((B, m.D, m.N))) for _ in m.blocks]

    def cn_norm(x, g, res):
        if res is None:
            res = cnp.zeros(x.shape, dtype=dtype)
        return cnp.rms_norm(x, g, res), res

    # a product gives (tokens, features); a prompt of B sequences is laid out (B, n, .) by copies
    def rows3(x, B, n):
        out = cnp.empty((B, n, x.shape[1]), dtype=dtype)
        for b in range(B):
            out[b] = x[b * n:(b + 1) * n, :]
        return out

    def rows2(x, B, n):
        out = cnp.empty((B * n, x.shape[2]), dtype=dtype)
        for b in range(B):
            out[b * n:(b + 1) * n, :] = x[b, :, :]
        return out

    def cn_conv(xz, blk, st, B, n, D):
        if n == 1:
            return cnp.short_convolution(xz[:, :D], blk["conv"], blk["bias"], st["conv"])
        return rows2(cnp.short_convolution(rows3(xz, B, n)[:, :, :D], blk["conv"], blk["bias"], st["conv"]), B, n)

    def cn_scan(c, par, xz, blk, st, B, n, D, N):
        if n > 1:
            c, par, xz = (rows3(v, B, n) for v in (c, par, xz))
        at = (slice(None),) * (2 if n > 1 else 1)
        y = cnp.state_scan(c, par[at + (slice(0, D),)], blk["A"], par[at + (slice(D, D + N),)],
                           par[at + (slice(D + N, D + 2 * N),)], blk["skip"], xz[at + (slice(D, 2 * D),)], blk["db"], st["h"])
        return rows2(y, B, n) if n > 1 else y

    dev = [{k: cnp.array(v) for k, v in b.items()} for b in m.blocks]
    host = [dict(b) for b in m.blocks]
    dev[-1]["head"], host[-1]["head"] = cnp.array(m.head), m.head
    ds, hs = fresh(lambda s: cnp.zeros(s, dtype=dtype)), fresh(np.zeros)
    count, x = n, m.embed[words.reshape(-1)]
    seen = [words]
    for step in range(steps):
        want = forward(m, host, x, hs, B, count, np_norm, np_conv, np_scan, lambda a, b: a @ b)
        logits = forward(m, dev, cnp.array(x), ds, B, count, cn_norm, cn_conv, cn_scan, lambda a, b: a @ b)
        got = logits.get(itf)
        # everything is smooth and of size 1 to 100: rounding differences of 2^-53 stay far below 1e-10
        assert np.abs(got - want).max() <= 1e-10 * np.abs(want).max(), step
        last = want.reshape(B, count, m.V)[:, -1]
        if count > 1:
            final = cnp.empty((B, m.V), dtype=dtype)
            for b in range(B):
                final[b:b + 1, :] = logits[(b + 1) * count - 1:(b + 1) * count, :]
        else:
            final = logits
        drawn = cnp.random.sample_tokens(final, us[step], 0.9, 40, 0.95).get(itf)
        for b in range(B):
            word, near = R.sample_tokens(last[b], us[step, b], 0.9, 40, 0.95, 0.0)
            assert near < 1e-8 or drawn[b] == word, (step, b)
        seen.append(drawn[:, None])
        count, x = 1, m.embed[drawn]
    for a, b in zip(ds, hs):
        assert np.abs(a["h"].get(itf) - b["h"]).max() <= 1e-10 and np.abs(a["conv"].get(itf) - b["conv"]).max() <= 1e-10
    whole = np.concatenate(seen[:-1], axis=1)
    again = forward(m, dev, cnp.array(m.embed[whole.reshape(-1)]), fresh(lambda s: cnp.zeros(s, dtype=dtype)), B,
                    whole.shape[1], cn_norm, cn_conv, cn_scan, lambda a, b: a @ b).get(itf)
    assert np.abs(again.reshape(B, -1, m.V)[:, -1] - last).max() <= 1e-10 * np.abs(last).max()


def test_results_go_on_into_statements_and_products(itf):
    """What a call returns is an array like any other, and what it updates is seen by what follows."""
    rng = np.random.default_rng(0)
    x, r = rng.standard_normal((24, 32)), rng.standard_normal((24, 32))
    w = rng.standard_normal((32, 16))
    dx, dr = cnp.array(x), cnp.array(r)
    before = dr * 2.0
    y = cnp.rms_norm(dx + 1.0, residual=dr)
    out = (y * 0.5) @ cnp.array(w) + 1.0
    twice = dr - before * 0.5
    total = cnp.sum(y)
    s = x + 1.0 + r
    n = s / np.sqrt((s * s).mean(axis=1, keepdims=True) + 1e-6)
    assert np.allclose(out.get(itf), (n * 0.5) @ w + 1.0, rtol=1e-12, atol=1e-12)
    assert np.allclose(twice.get(itf), x + 1.0, rtol=1e-13, atol=1e-13)
    assert np.allclose(total.get(itf), n.sum(), rtol=1e-11)
    ones = cnp.ones((8,))
    cnp.rms_norm(cnp.array(np.arange(8.0)), residual=ones)     # no longer all ones: a dot has to read it
    assert np.allclose(ones.dot(cnp.array(np.ones(8))).get(itf), 36.0)
