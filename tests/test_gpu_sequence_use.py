"""The sequence operators' C entry points the way a server uses them: captured into a graph, on streams of
their own, at offsets beyond 32 bits, with more sequences than a grid holds, without an allocation."""
import ctypes as C

import numpy as np
import pytest

from charmnumeric_amd import _lib as L
from tests import helpers as H
from tests import sequence_reference as R
from tests.test_gpu_sequence import close, scan_call, scan_inputs

pytestmark = pytest.mark.gpu


class Step:
    """norm -> convolution -> scan -> draw on torch tensors, every buffer kept: one call queues it all."""

    def __init__(self, torch, B, n, D, N=16, K=4, seed=0):
        self.torch, self.dims = torch, (B, n, D, N, K)
        g = torch.Generator(device="cuda").manual_seed(seed)
        f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.x, self.res, self.g = f(B * n, D), f(B * n, D), 1 + 0.1 * f(D)
        self.h, self.conv_state, self.state = f(B * n, D), f(B, K - 1, D), f(B, D, N)
        self.w, self.bias, self.delta, self.z = f(K, D), f(D), 0.5 * f(B, n, D), f(B, n, D)
        self.A = -torch.arange(1.0, N + 1, device="cuda").repeat(D, 1)
        self.Bm, self.Cm, self.skip, self.db = f(B, n, N), f(B, n, N), f(D), f(D) - 4
        self.c, self.y = f(B, n, D), f(B, n, D)
        self.u = torch.rand(B, generator=g, device="cuda", dtype=torch.float64)
        self.words = torch.zeros(B, device="cuda", dtype=torch.int32)
        self.space = None
        self.scan = self.scan_args()
        need = L.check(L.lib.cnh_state_scan_workspace(C.byref(self.scan)))
        if need:
            self.space = torch.empty(need, device="cuda", dtype=torch.uint8)
            self.scan.workspace, self.scan.workspace_bytes = self.space.data_ptr(), need

    def scan_args(self):
        B, n, D, N, K = self.dims
        p = lambda t: t.data_ptr()  # noqa: E731
        return L.StateScan(L.F32, 1, B, n, D, N, p(self.c), n * D, D, p(self.delta), n * D, D, p(self.z), n * D, D,
                           p(self.A), p(self.Bm), n * N, N, p(self.Cm), n * N, N, p(self.skip), p(self.db), p(self.state),
                           p(self.state), None, p(self.y), n * D, D)

    def __call__(self):
        B, n, D, N, K = self.dims
        p = lambda t: t.data_ptr()  # noqa: E731
        s = self.torch.cuda.current_stream().cuda_stream
        L.check(L.lib.cnh_rms_norm(C.byref(L.RmsNorm(L.F32, B * n, D, p(self.x), D, p(self.res), D, p(self.res), D,
                                                     p(self.g), 1e-6, p(self.h), D)), s))
        L.check(L.lib.cnh_short_convolution(C.byref(L.ShortConvolution(
            L.F32, 1, K, B, n, D, p(self.h), n * D, D, p(self.w), p(self.bias), p(self.conv_state), p(self.conv_state),
            None, p(self.c), n * D, D)), s))
        L.check(L.lib.cnh_state_scan(C.byref(self.scan), s))
        a = L.SampleTokens(L.F32, 20, B, D, p(self.y) + (n - 1) * D * 4, n * D, p(self.u), 0.7, 0.9, 0.0)
        a.out = p(self.words)
        L.check(L.lib.cnh_sample_tokens(C.byref(a), s))

    def carried(self):
        return [t.clone() for t in (self.res, self.conv_state, self.state)]

    def results(self):
        return [t.cpu().numpy() for t in (self.res, self.h, self.c, self.conv_state, self.y, self.state, self.words)]


@pytest.fixture(scope="module")
def torch():
    t = pytest.importorskip("torch")
    L.check(L.lib.cnh_init(0))
    return t


@pytest.mark.parametrize("B,n,D", [(3, 1, 320), (1, 600, 128), (2, 40, 256)])
def test_captured_and_replayed(torch, B, n, D):
    """A captured step, replayed with eager steps and synchronisations between, carries the states on
    exactly as eager steps do; the launches of a call do not depend on where it is recorded."""
    one, two = Step(torch, B, n, D), Step(torch, B, n, D)
    other = Step(torch, B, n, D, seed=9)
    assert one.space is not None or n < 600           # the long prompt is cut, with a workspace
    one()
    two()
    torch.cuda.synchronize()
    before = one.carried()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    for t, v in zip((one.res, one.conv_state, one.state), before):
        assert torch.equal(t, v)                     # recording ran nothing
    for k in range(4):
        one.x.normal_()                              # new input, the same buffers
        two.x.copy_(one.x)
        graph.replay()
        other()
        two()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(one.results(), two.results())):
            assert np.array_equal(a, b), (k, i)


def test_two_streams_at_once(torch):
    """Calls on two streams, each with buffers and a workspace of its own, give what they give alone."""
    steps = [Step(torch, 1, 600, 128, seed=s) for s in (1, 2)]
    alone = [Step(torch, 1, 600, 128, seed=s) for s in (1, 2)]
    for s in alone:
        for _ in range(5):
            s()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                s()
    torch.cuda.synchronize()
    for a, b in zip(steps, alone):
        for u, v in zip(a.results(), b.results()):
            assert np.array_equal(u, v)


def test_calls_allocate_nothing(torch):
    s = Step(torch, 1, 600, 128)
    s()
    torch.cuda.synchronize()
    before = L.lib.cnh_allocation_count()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(3):
        s()
    torch.cuda.synchronize()
    assert L.lib.cnh_allocation_count() == before and torch.cuda.mem_get_info()[0] == free


def far_apart(dev, rows, stride, dtype=np.float32):
    """Rows of one array `stride` elements apart in a buffer that is not written elsewhere."""
    p = C.c_void_p()
    bytes_ = (stride * (len(rows) - 1) + rows[0].size) * np.dtype(dtype).itemsize
    L.check(L.lib.cnh_alloc(bytes_, 0, C.byref(p)))
    for i, r in enumerate(rows):
        r = np.ascontiguousarray(r, dtype)
        L.check(L.lib.cnh_h2d(p.value + i * stride * r.itemsize, r.ctypes.data, r.nbytes, None))
    return p.value


def fetch(ptr, stride, shape, count, dtype=np.float32):
    out = []
    for i in range(count):
        a = np.empty(shape, dtype)
        L.check(L.lib.cnh_d2h(a.ctypes.data, ptr + i * stride * a.itemsize, a.nbytes, None))
        out.append(a)
    return np.stack(out)


FAR = 2_200_000_000        # elements: beyond 2^31 elements and 2^33 bytes


def test_offsets_beyond_32_bits(dev):
    rng = np.random.default_rng(0)
    u = R.half_step(np.float32)
    x = rng.standard_normal((3, 1000)).astype(np.float32)
    px, py = far_apart(dev, x, FAR), far_apart(dev, np.zeros_like(x), FAR)
    L.check(L.lib.cnh_rms_norm(C.byref(L.RmsNorm(L.F32, 3, 1000, px, FAR, None, 0, None, 0, None, 1e-6, py, FAR)), None))
    y, _, ey, _ = R.rms_norm(x, None, None, 1e-6, u)
    close(fetch(py, FAR, 1000, 3), y, ey, "norm")

    logits, un = x * 3, rng.random(3)
    du, out = dev.array(un), dev.array(np.zeros(3, np.int32))
    for i in range(3):
        L.check(L.lib.cnh_h2d(px + i * FAR * 4, np.ascontiguousarray(logits[i]).ctypes.data, 4000, None))
    a = L.SampleTokens(L.F32, 0, 3, 1000, px, FAR, du.ptr, 1.0, 0.9, 0.0)
    a.out = out.ptr
    L.check(L.lib.cnh_sample_tokens(C.byref(a), None))
    assert out.get().tolist() == [R.sample_tokens(logits[i], un[i], 1.0, 0, 0.9, 0.0)[0] for i in range(3)]
    for p in (px, py):
        L.check(L.lib.cnh_free(p))

    B, n, D, N, K = 3, 20, 64, 16, 4
    q = scan_inputs(np.float32, B, n, D, N, 1)
    w = rng.standard_normal((K, D)).astype(np.float32)
    px, py = far_apart(dev, q["x"], FAR), far_apart(dev, np.zeros_like(q["x"]), FAR)
    dw = dev.array(w)
    L.check(L.lib.cnh_short_convolution(C.byref(L.ShortConvolution(
        L.F32, 1, K, B, n, D, px, FAR, D, dw.ptr, None, None, None, None, py, FAR, D)), None))
    y, _, ey = R.short_convolution(q["x"], w, None, None, None, True, u)
    close(fetch(py, FAR, (n, D), B), y, ey, "convolution")
    d = {k: dev.array(v) for k, v in q.items()}
    hs = dev.array(np.zeros((B, D, N), np.float32))
    a = L.StateScan(L.F32, 1, B, n, D, N, px, FAR, D, d["delta"].ptr, n * D, D, d["z"].ptr, n * D, D, d["A"].ptr,
                    d["Bm"].ptr, n * N, N, d["Cm"].ptr, n * N, N, d["skip"].ptr, d["delta_bias"].ptr, d["state"].ptr, hs.ptr,
                    None, py, FAR, D)
    need = L.check(L.lib.cnh_state_scan_workspace(C.byref(a)))
    if need:
        ws = dev.array(np.zeros(need, np.uint8))
        a.workspace, a.workspace_bytes = ws.ptr, need
    L.check(L.lib.cnh_state_scan(C.byref(a), None))
    y, h, ey, eh = R.state_scan(**q, lengths=None, softplus=True, u=u, piece=64)
    close(fetch(py, FAR, (n, D), B), y, ey, "scan")
    close(hs.get(), h, eh, "state")
    for p in (px, py):
        L.check(L.lib.cnh_free(p))
    dev.free_all()


def test_more_sequences_and_rows_than_a_grid_holds(dev):
    """70000 sequences through the convolution and the scan (prompts and tokens), a million rows and more
    through the norm and the draw: one row repeated by a stride of zero where it is only read."""
    u = R.half_step(np.float32)
    B, D, N, K = 70_000, 5, 4, 3
    for n in (2, 1):
        q = scan_inputs(np.float32, 1, n, D, N, 3)
        rep = dev.array(np.repeat(q["state"], B, axis=0))
        one = {k: dev.array(v) for k, v in q.items()}
        dy = dev.array(np.full((B, n, D), 7, np.float32))
        a = L.StateScan(L.F32, 1, B, n, D, N, one["x"].ptr, 0, D, one["delta"].ptr, 0, D, one["z"].ptr, 0, D, one["A"].ptr,
                        one["Bm"].ptr, 0, N, one["Cm"].ptr, 0, N, one["skip"].ptr, one["delta_bias"].ptr, rep.ptr, rep.ptr,
                        None, dy.ptr, n * D, D)
        assert L.lib.cnh_state_scan_workspace(C.byref(a)) == 0
        L.check(L.lib.cnh_state_scan(C.byref(a), None))
        y, h, ey, eh = R.state_scan(**q, lengths=None, softplus=True, u=u)
        got, hs = dy.get(), rep.get()
        assert (got == got[:1]).all() and (hs == hs[:1]).all()
        close(got[:1], y, ey, "scan")
        close(hs[:1], h, eh, "state")
        w = np.random.default_rng(1).standard_normal((K, D)).astype(np.float32)
        dw, st = dev.array(w), dev.array(np.zeros((B, K - 1, D), np.float32))
        L.check(L.lib.cnh_short_convolution(C.byref(L.ShortConvolution(
            L.F32, 0, K, B, n, D, one["x"].ptr, 0, D, dw.ptr, None, st.ptr, st.ptr, None, dy.ptr, n * D, D)), None))
        y, after, ey = R.short_convolution(q["x"], w, None, np.zeros((1, K - 1, D)), None, False, u)
        got, st = dy.get(), st.get()
        assert (got == got[:1]).all() and (st == st[:1]).all()
        close(got[:1], y, ey, "convolution")
        assert np.array_equal(st[:1].astype(np.float64), after)
        dev.free_all()
    rows, cols = (1 << 20) + 3, 1028
    x = np.random.default_rng(2).standard_normal((1, cols)).astype(np.float32)
    dx = dev.array(x)
    p = C.c_void_p()
    L.check(L.lib.cnh_alloc(rows * cols * 4, 1, C.byref(p)))
    L.check(L.lib.cnh_rms_norm(C.byref(L.RmsNorm(L.F32, rows, cols, dx.ptr, 0, None, 0, None, 0, None, 1e-6, p.value, cols)),
                               None))
    y, _, ey, _ = R.rms_norm(x, None, None, 1e-6, u)
    for first in (0, 1 << 19, (1 << 20) - 1, rows - 3):
        got = fetch(p.value + first * cols * 4, cols, cols, 3)
        close(got, np.repeat(y, 3, axis=0), np.repeat(ey, 3, axis=0), f"norm, rows from {first}")
    L.check(L.lib.cnh_free(p))
    n, D, K = 4 * 65535 * 8 + 21, 3, 3                       # one long sequence through the convolution
    x = np.random.default_rng(4).standard_normal((1, n, D)).astype(np.float32)
    w = np.random.default_rng(5).standard_normal((K, D)).astype(np.float32)
    dx, dw, dy, st = dev.array(x), dev.array(w), dev.array(np.full((1, n, D), 7, np.float32)), dev.array(np.zeros((1, K - 1, D), np.float32))
    L.check(L.lib.cnh_short_convolution(C.byref(L.ShortConvolution(
        L.F32, 0, K, 1, n, D, dx.ptr, n * D, D, dw.ptr, None, None, st.ptr, None, dy.ptr, n * D, D)), None))
    y, after, ey = R.short_convolution(x, w, None, None, None, False, u)
    close(dy.get(), y, ey, "convolution of a long sequence")
    assert np.array_equal(st.get().astype(np.float64), after)
    dev.free_all()
    logits = dev.array(np.array([0.0, 1.0, 2.0, -1.0], np.float32))
    un = np.random.default_rng(3).random(rows)
    du, out = dev.array(un), dev.array(np.full(rows, -9, np.int32))
    a = L.SampleTokens(L.F32, 0, rows, 4, logits.ptr, 0, du.ptr, 1.0, 1.0, 0.0)
    a.out = out.ptr
    L.check(L.lib.cnh_sample_tokens(C.byref(a), None))
    w = np.exp(np.array([2.0, 1.0, 0.0, -1.0]))              # in descending order: words 2, 1, 0, 3
    upto = np.cumsum(w) / w.sum()
    place = np.searchsorted(upto, un, side="right")
    clear = np.abs(un[:, None] - upto).min(axis=1) > 1e-12
    assert np.array_equal(out.get()[clear], np.array([2, 1, 0, 3])[np.minimum(place, 3)][clear])
    dev.free_all()


def test_padding_and_memory_behind_the_sequences(dev):
    """Padded rows are zeros, memory between rows that are apart stays as it was, and what a call reads is
    not written."""
    B, n, D, N = 3, 9, 40, 16
    q = scan_inputs(np.float32, B, n, D, N, 5)
    d = {k: dev.array(v) for k, v in q.items()}
    lengths = dev.array(np.array([4, 0, 9], np.int32))
    dy = dev.array(np.full((B, n + 2, D + 3), 5, np.float32))
    h = dev.array(np.zeros((B, D, N), np.float32))
    a = L.StateScan(L.F32, 1, B, n, D, N, d["x"].ptr, n * D, D, d["delta"].ptr, n * D, D, d["z"].ptr, n * D, D, d["A"].ptr,
                    d["Bm"].ptr, n * N, N, d["Cm"].ptr, n * N, N, d["skip"].ptr, d["delta_bias"].ptr, d["state"].ptr, h.ptr,
                    lengths.ptr, dy.ptr, (n + 2) * (D + 3), D + 3)
    L.check(L.lib.cnh_state_scan(C.byref(a), None))
    got = dy.get()
    for b, k in enumerate((4, 0, 9)):
        assert (got[b, k:n, :D] == 0).all() and (got[b, :k, :D] != 0).any(axis=1).all()
        assert (got[b, :, D:] == 5).all() and (got[b, n:] == 5).all()
    assert np.array_equal(h.get()[1], q["state"][1])
    for k, v in q.items():
        assert np.array_equal(d[k].get(), v), k
    dev.free_all()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("B,n,N", [
    (2048, 33, 5), (2048, 33, 8), (2048, 33, 12), (2048, 33, 16), (2048, 33, 20), (2048, 33, 32), (2048, 33, 40),
    (256, 256, 5), (256, 256, 8), (256, 256, 12), (256, 256, 16), (256, 256, 20), (256, 256, 32),
    (600, 130, 6), (600, 130, 12), (600, 130, 16), (600, 130, 32), (700, 130, 7), (700, 130, 16), (700, 130, 24),
])
def test_scan_of_many_sequences(dev, dtype, B, n, N):
    """Batches that fill the device, with one and with several states a lane, whole and cut: one sequence
    repeated by a stride of zero, every one of them with a state of its own."""
    D, u = 64, R.half_step(dtype)
    q = scan_inputs(dtype, 1, n, D, N, n + N)
    one, rep = {k: dev.array(v) for k, v in q.items()}, dev.array(np.repeat(q["state"], B, axis=0))
    dy = dev.array(np.full((B, n, D), 7, dtype))
    a = L.StateScan(L.F32 if dtype == np.float32 else L.F64, 1, B, n, D, N, one["x"].ptr, 0, D, one["delta"].ptr, 0, D,
                    one["z"].ptr, 0, D, one["A"].ptr, one["Bm"].ptr, 0, N, one["Cm"].ptr, 0, N, one["skip"].ptr,
                    one["delta_bias"].ptr, rep.ptr, rep.ptr, None, dy.ptr, n * D, D)
    a.workspace_bytes = L.check(L.lib.cnh_state_scan_workspace(C.byref(a)))
    if a.workspace_bytes:
        a.workspace = dev.array(np.full(a.workspace_bytes // 4, np.nan, np.float32)).ptr
    L.check(L.lib.cnh_state_scan(C.byref(a), None))
    y, h, ey, eh = R.state_scan(**q, lengths=None, softplus=True, u=u, piece=64)
    got, hs = dy.get(), rep.get()
    assert (got == got[:1]).all() and (hs == hs[:1]).all()
    close(got[:1], y, ey, "scan")
    close(hs[:1], h, eh, "state")
    dev.free_all()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("n,N", [(1, 16), (40, 16), (40, 13), (40, 100), (700, 8)])
def test_scan_of_infinities_and_nan(dev, dtype, n, N):
    """A rate of -infinity forgets at once, whatever came before; what is no number stays in its channel and
    behind its token. The longest prompt is padded by more than a piece of its cut."""
    D, u = 70, R.half_step(dtype)
    last = n if n < 700 else n - 50
    lengths = None if last == n else [last]
    q = scan_inputs(dtype, 1, n, D, N, n * N)
    q["A"][:, 0] = -1e6                                       # decays that are zero already
    q["delta_bias"][:] = 1.0                                  # steps of 0.1 and more
    y, h, ey, eh = R.state_scan(**q, lengths=lengths, softplus=True, u=u, piece=64)
    q["A"][:, 0] = -np.inf
    bad = n // 2
    q["x"][0, bad, 5] = np.nan
    q["delta"][0, bad, 66] = np.nan
    q["A"][9, N - 1] = np.nan
    q["z"][0, bad, 12] = np.nan
    got, out, _ = scan_call(dev, dtype, q, lengths, True)
    for d in (5, 66, 9):
        first = 0 if d == 9 else bad
        assert np.isnan(got[0, first:last, d]).all()
        assert np.isnan(out[0, d]).all() if d != 9 else np.isnan(out[0, d, N - 1])
        got[0, first:last, d], out[0, d] = y[0, first:last, d], h[0, d]
    assert np.isnan(got[0, bad, 12])
    got[0, bad, 12] = y[0, bad, 12]
    close(got, y, ey, "scan")
    close(out, h, eh, "state")
    dev.free_all()
