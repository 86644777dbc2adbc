"""Timed cases of the sequence operators: root-mean-square norm with the residual's addition, the
short causal convolution and the selective state space scan of a recurrent block (for prompts and
for single tokens), and the draw of the next token from its logits.

`run` computes a case in elementary torch operations, or, where `own` is true, through the C entry
points of charmnumeric_amd (include/cnhip.h) on torch's stream.
"""
import torch

own = False

_TYPES = {"f32": torch.float32, "f64": torch.float64}
_MEMORY = 34_000_000      # elements of the largest tensor of a drawn case


def listed():
    return [
        # one decoding step of a small batch: the launch is what it costs
        dict(name="norm_token", op="norm", type="f32", rows=4, cols=1024, residual=True),
        # a long prompt, the residual stream updated on the way
        dict(name="norm_prompt", op="norm", type="f32", rows=16384, cols=2048, residual=True),
        # odd width in double precision, the norm in front of the head (no residual)
        dict(name="norm_odd_f64", op="norm", type="f64", rows=777, cols=1537, residual=False),
        # a batch of long prompts through the four-tap convolution
        dict(name="conv_prompt", op="conv", type="f32", batch=4, length=2048, channels=4096, taps=4, silu=True,
             ragged=False),
        # prompts of different lengths padded into one batch, double precision
        dict(name="conv_ragged_f64", op="conv", type="f64", batch=7, length=333, channels=1100, taps=3, silu=False,
             ragged=True),
        # one decoding step of 64 sequences
        dict(name="conv_token", op="conv", type="f32", batch=64, length=1, channels=4096, taps=4, silu=True,
             ragged=False),
        # one long prompt alone on the card
        dict(name="scan_prompt", op="scan", type="f32", batch=1, length=8192, channels=2048, states=16, ragged=False),
        # padded prompts of different lengths, a width that is no multiple of a wavefront
        dict(name="scan_ragged", op="scan", type="f32", batch=6, length=1111, channels=1000, states=16, ragged=True),
        # a short run in double precision, as a check of a single-precision model
        dict(name="scan_f64", op="scan", type="f64", batch=2, length=500, channels=512, states=8, ragged=False),
        # one decoding step of 128 sequences: the states are read and written once
        dict(name="scan_token", op="scan", type="f32", batch=128, length=1, channels=4096, states=16, ragged=False),
        # the next token of one sequence, a large vocabulary
        dict(name="sample_one", op="sample", type="f32", rows=1, vocab=131072, per_row=False, top_k=50, top_p=0.95,
             min_p=0.0, temperature=0.8),
        # the next tokens of 256 sequences, every one with settings of its own
        dict(name="sample_batch", op="sample", type="f32", rows=256, vocab=50021, per_row=True, top_k=200,
             top_p=0.9, min_p=0.01, temperature=1.0),
    ]


def _log_between(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "conv", "scan", "sample"])
    kind = rng.choice(["f32", "f32", "f64"])
    if op == "norm":
        cols = _log_between(rng, 64, 8192)
        rows = _log_between(rng, 1, min(16384, _MEMORY // 2 // cols))
        return dict(op=op, type=kind, rows=rows, cols=cols, residual=rng.random() < 0.7)
    if op == "conv":
        batch, channels = _log_between(rng, 1, 64), _log_between(rng, 64, 4096)
        length = 1 if rng.random() < 0.3 else _log_between(rng, 2, max(2, min(8192, _MEMORY // 2 // (batch * channels))))
        return dict(op=op, type=kind, batch=batch, length=length, channels=channels, taps=rng.randint(2, 4),
                    silu=rng.random() < 0.7, ragged=length > 1 and rng.random() < 0.5)
    if op == "scan":
        batch, channels = _log_between(rng, 1, 128), _log_between(rng, 64, 4096)
        states = rng.choice([4, 8, 13, 16, 16, 16, 32])
        most = max(2, min(8192, 4_000_000 * 16 // (batch * channels * states)))
        length = 1 if rng.random() < 0.3 else _log_between(rng, 2, most)
        return dict(op=op, type=kind, batch=batch, length=length, channels=channels, states=states,
                    ragged=length > 1 and rng.random() < 0.5)
    vocab = _log_between(rng, 1000, 131072)
    rows = _log_between(rng, 1, min(256, 12_800_000 // vocab))
    return dict(op=op, type=kind, rows=rows, vocab=vocab, per_row=rng.random() < 0.5,
                top_k=rng.choice([0, 0, 1, 20, 50, 300, 2000]), top_p=rng.choice([1.0, 0.9, 0.95, 0.5]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), temperature=rng.choice([0.0, 0.7, 1.0, 1.3]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    T = _TYPES[case["type"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=T).mul_(scale)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64).mul_(hi - lo).add_(lo)

    s = dict(case)
    if case["op"] == "norm":
        s["x"] = randn(case["rows"], case["cols"])
        s["res"] = randn(case["rows"], case["cols"], scale=3.0) if case["residual"] else None
        s["weight"] = 1.0 + randn(case["cols"], scale=0.1)
        return s
    if case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        logits = randn(R, V, scale=2.5)
        # words that the grammar or the user has ruled out
        logits[torch.rand(R, V, generator=g, device="cuda") < 0.05] = float("-inf")
        s["logits"], s["u"] = logits, uniform(R)
        if case["per_row"]:
            s["temperatures"] = case["temperature"] * uniform(R, lo=0.5, hi=1.5)
            s["top_ks"] = torch.randint(0, 2 * case["top_k"] + 1, (R,), generator=g, device="cuda", dtype=torch.int32)
            s["top_ps"] = case["top_p"] * uniform(R, lo=0.8, hi=1.1)
            s["min_ps"] = case["min_p"] * uniform(R, lo=0.0, hi=2.0)
        return s
    B, L, D = case["batch"], case["length"], case["channels"]
    lengths = torch.randint(0, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    s["lengths"] = lengths if case["ragged"] else None
    # a block's input and its gate leave one projection side by side
    xz = randn(B, L, 2 * D)
    if case["op"] == "conv":
        K = case["taps"]
        s["x"] = xz[:, :, :D]
        s["weight"], s["bias"] = randn(K, D, scale=0.5), randn(D, scale=0.1)
        s["state"] = randn(B, K - 1, D)
        return s
    N = case["states"]
    s["x"], s["z"] = randn(B, L, D), xz[:, :, D:]
    s["delta"] = randn(B, L, D, scale=0.5)
    # steps of 0.001 to 0.1 behind the softplus; decay rates around 1..N
    s["delta_bias"] = torch.log(torch.expm1(torch.exp(uniform(D, lo=-6.9, hi=-2.3)))).to(T)
    rates = torch.arange(1, N + 1, device="cuda", dtype=T).expand(D, N)
    s["A"] = -(rates * torch.exp(randn(D, N, scale=0.1)))
    bc = randn(B, L, 2 * N)
    s["B"], s["C"] = bc[:, :, :N], bc[:, :, N:]
    s["skip"] = 1.0 + randn(D, scale=0.1)
    s["state"] = randn(B, D, N)
    return s


# ---- the plain forms ------------------------------------------------------------------------------


def _plain_norm(s):
    r = s["x"] + s["res"] if s["residual"] else s["x"]
    y = r * torch.rsqrt(r.square().mean(dim=1, keepdim=True) + 1e-6) * s["weight"]
    return (y, r) if s["residual"] else (y,)


def _within(s):
    """(batch, length) truth values: does the token belong to its sequence?"""
    return torch.arange(s["length"], device="cuda")[None, :] < s["lengths"][:, None]


def _plain_conv(s):
    B, L, D, K = s["batch"], s["length"], s["channels"], s["taps"]
    ext = torch.cat([s["state"], s["x"]], dim=1)
    y = (ext.unfold(1, L, 1) * s["weight"][None, :, :, None]).sum(dim=1).transpose(1, 2) + s["bias"]
    if s["silu"]:
        y = y / (1.0 + torch.exp(-y))
    if s["lengths"] is None:
        return y.contiguous(), ext[:, L:].contiguous()
    at = s["lengths"].long()[:, None] + torch.arange(K - 1, device="cuda")[None, :]
    state = torch.gather(ext, 1, at[:, :, None].expand(B, K - 1, D))
    return torch.where(_within(s)[:, :, None], y, 0.0), state


def _plain_scan(s):
    x, n = s["x"], s["length"]
    step = s["delta"] + s["delta_bias"]
    step = torch.where(step > 20.0, step, torch.log1p(torch.exp(step)))
    if s["lengths"] is not None:
        # a step of zero leaves the state as it is
        step = torch.where(_within(s)[:, :, None], step, 0.0)
    a = torch.exp(step[..., None] * s["A"])
    h = (step * x)[..., None] * s["B"][:, :, None, :]
    h[:, 0] += a[:, 0] * s["state"]
    # h_t = a_t h_(t-1) + b_t by doubling: after the pass with distance d each h_t holds 2 d terms
    d = 1
    while d < n:
        h = torch.cat([h[:, :d], h[:, d:] + a[:, d:] * h[:, :-d]], dim=1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], dim=1)
        d *= 2
    y = (h * s["C"][:, :, None, :]).sum(dim=3) + s["skip"] * x
    y = y * s["z"] / (1.0 + torch.exp(-s["z"]))
    if s["lengths"] is not None:
        y = torch.where(_within(s)[:, :, None], y, 0.0)
    return y, h[:, -1].contiguous()


def _settings(s):
    R = s["rows"]
    if s["per_row"]:
        return s["temperatures"], s["top_ks"].long(), s["top_ps"], s["min_ps"]
    full = lambda v, t: torch.full((R,), v, device="cuda", dtype=t)  # noqa: E731
    return (full(s["temperature"], torch.float64), full(s["top_k"], torch.int64), full(s["top_p"], torch.float64),
            full(s["min_p"], torch.float64))


def _plain_sample(s):
    # in 64 bits: the drawn word changes where the running sum passes the random number
    temperature, top_k, top_p, min_p = _settings(s)
    V = s["vocab"]
    logits = s["logits"].double()
    top, best = logits.max(dim=1)
    w = torch.exp((logits - top[:, None]) / temperature[:, None])
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    sorted_w = torch.gather(w, 1, order)
    rank = torch.arange(V, device="cuda")[None, :]
    keep = (top_k[:, None] <= 0) | (rank < top_k[:, None])
    sorted_w = torch.where(keep, sorted_w, 0.0)
    before = sorted_w.cumsum(dim=1) - sorted_w
    total = sorted_w.sum(dim=1, keepdim=True)
    keep &= (top_p[:, None] >= 1.0) | (before < top_p[:, None] * total)
    keep &= sorted_w >= min_p[:, None]
    upto = torch.where(keep, sorted_w, 0.0).cumsum(dim=1)
    place = (upto <= s["u"][:, None] * upto[:, -1:]).sum(dim=1).clamp(max=V - 1)
    drawn = torch.gather(order, 1, place[:, None])[:, 0]
    return torch.where(temperature > 0.0, drawn, best).int()


# ---- through the framework ------------------------------------------------------------------------


def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    import ctypes

    from charmnumeric_amd import _lib as L
    stream = torch.cuda.current_stream().cuda_stream
    dt = L.F32 if s["type"] == "f32" else L.F64
    op = s["op"]
    if op == "norm":
        x, res = s["x"], s["res"]
        rows, cols = x.shape
        y = torch.empty_like(x)
        out = torch.empty_like(x) if s["residual"] else None
        L.check(L.lib.cnh_rms_norm(ctypes.byref(L.RmsNorm(
            dt, rows, cols, x.data_ptr(), cols, _p(res), cols, _p(out), cols, s["weight"].data_ptr(), 1e-6,
            y.data_ptr(), cols)), stream))
        return (y, out) if s["residual"] else (y,)
    if op == "conv":
        x, state = s["x"], s["state"]
        B, n, D = x.shape
        y = torch.empty((B, n, D), device=x.device, dtype=x.dtype)
        out = torch.empty_like(state)
        L.check(L.lib.cnh_short_convolution(ctypes.byref(L.ShortConvolution(
            dt, 1 if s["silu"] else 0, s["taps"], B, n, D, x.data_ptr(), x.stride(0), x.stride(1),
            s["weight"].data_ptr(), s["bias"].data_ptr(), state.data_ptr(), out.data_ptr(), _p(s["lengths"]),
            y.data_ptr(), n * D, D)), stream))
        return y, out
    if op == "scan":
        x, delta, z, b, c, state = s["x"], s["delta"], s["z"], s["B"], s["C"], s["state"]
        B, n, D = x.shape
        y = torch.empty((B, n, D), device=x.device, dtype=x.dtype)
        out = torch.empty_like(state)
        args = L.StateScan(
            dt, 1, B, n, D, s["states"], x.data_ptr(), x.stride(0), x.stride(1), delta.data_ptr(), delta.stride(0),
            delta.stride(1), z.data_ptr(), z.stride(0), z.stride(1), s["A"].data_ptr(), b.data_ptr(), b.stride(0),
            b.stride(1), c.data_ptr(), c.stride(0), c.stride(1), s["skip"].data_ptr(), s["delta_bias"].data_ptr(),
            state.data_ptr(), out.data_ptr(), _p(s["lengths"]), y.data_ptr(), n * D, D)
        need = L.check(L.lib.cnh_state_scan_workspace(ctypes.byref(args)))
        if need:
            space = torch.empty(need, device=x.device, dtype=torch.uint8)
            args.workspace, args.workspace_bytes = space.data_ptr(), need
        L.check(L.lib.cnh_state_scan(ctypes.byref(args), stream))
        return y, out
    logits = s["logits"]
    R, V = logits.shape
    out = torch.empty(R, device=logits.device, dtype=torch.int32)
    args = L.SampleTokens(dt, s["top_k"], R, V, logits.data_ptr(), V, s["u"].data_ptr(), s["temperature"], s["top_p"],
                          s["min_p"])
    if s["per_row"]:
        args.temperatures, args.top_ks = s["temperatures"].data_ptr(), s["top_ks"].data_ptr()
        args.top_ps, args.min_ps = s["top_ps"].data_ptr(), s["min_ps"].data_ptr()
    args.out = out.data_ptr()
    need = L.check(L.lib.cnh_sample_tokens_workspace(ctypes.byref(args)))
    if need:
        space = torch.empty(need, device=logits.device, dtype=torch.uint8)
        args.workspace, args.workspace_bytes = space.data_ptr(), need
    L.check(L.lib.cnh_sample_tokens(ctypes.byref(args), stream))
    return out


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan, "sample": _plain_sample}[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------


def work(case):
    e = 4 if case["type"] == "f32" else 8
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": e * (n * (4 if case["residual"] else 2) + case["cols"]),
                "flops": n * (5 if case["residual"] else 4)}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": e * n + case["rows"] * (12 + (28 if case["per_row"] else 0)), "flops": 2 * n}
    B, L, D = case["batch"], case["length"], case["channels"]
    n = B * L * D
    if case["op"] == "conv":
        K = case["taps"]
        return {"bytes": e * (2 * n + 2 * B * (K - 1) * D + (K + 1) * D), "flops": n * (2 * K + (4 if case["silu"] else 0))}
    N = case["states"]
    return {"bytes": e * (4 * n + 2 * B * L * N + 2 * B * D * N + D * N + 2 * D), "flops": n * (7 * N + 10)}


# ---- the definitions in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    up = lambda k: s[k].double()  # noqa: E731
    if case["op"] == "norm":
        r = up("x") + up("res") if case["residual"] else up("x")
        size = (r.pow(2).sum(dim=1) / case["cols"] + 1e-6).sqrt()
        y = r / size[:, None] * up("weight")
        return (y, r) if case["residual"] else (y,)
    if case["op"] == "sample":
        return None
    B, L, D = case["batch"], case["length"], case["channels"]
    ends = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    x = up("x")
    y = torch.zeros(B, L, D, device="cuda", dtype=torch.float64)
    if case["op"] == "conv":
        K, state, weight = case["taps"], up("state"), up("weight")
        last = torch.empty(B, K - 1, D, device="cuda", dtype=torch.float64)
        for b, n in enumerate(ends):
            rows = torch.cat([state[b], x[b, :n]])
            last[b] = rows[n:]
            for k in range(K):
                y[b, :n] += weight[k] * rows[k:k + n]
            y[b, :n] += up("bias")
            if case["silu"]:
                y[b, :n] *= torch.sigmoid(y[b, :n])
        return y, last
    if L > 20000:
        return None
    step = torch.logaddexp(up("delta") + up("delta_bias"), torch.zeros((), device="cuda", dtype=torch.float64))
    h, A, Bt, Ct = up("state").clone(), up("A"), up("B"), up("C")
    alive = torch.tensor(ends, device="cuda")
    for t in range(L):
        dt = step[:, t, :, None]
        new = h * torch.exp(dt * A) + dt * x[:, t, :, None] * Bt[:, t, None, :]
        here = (alive > t)[:, None]
        h = torch.where(here[..., None], new, h)
        y[:, t] = torch.where(here, torch.matmul(new, Ct[:, t, :, None])[..., 0], 0.0)
    z = up("z")
    inside = torch.arange(L, device="cuda")[None, :] < alive[:, None]
    y = torch.where(inside[..., None], (y + up("skip") * x) * z * torch.sigmoid(z), 0.0)
    return y, h
