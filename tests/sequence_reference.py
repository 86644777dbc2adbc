"""The sequence operators' definitions in NumPy, in 64 bits, each with a bound on what a kernel that
works in precision u (half a step of its type) may be off by, derived beside it. Used by the tests."""
import numpy as np


def half_step(dtype):
    return float(np.finfo(dtype).eps) / 2


def rms_norm(x, residual, weight, eps, u):
    x = x.astype(np.float64)
    r = x if residual is None else x + residual.astype(np.float64)
    n = r.shape[1]
    scale = 1.0 / np.sqrt((r * r).mean(axis=1, keepdims=True) + eps)
    y = r * scale * (1.0 if weight is None else weight.astype(np.float64))
    # r: one rounding. The sum of squares: a lane adds at most n / 64 + 8 terms and two trees add 10 more
    # levels, each term carries the squares' own roundings; half of that reaches the root. Root,
    # quotient, division by n and two products: 5 more.
    terms = n / 64 + 8 + 10 + 4
    return y, r, np.abs(y) * u * (1 + terms / 2 + 5 + 1), np.abs(r) * u


def short_convolution(x, weight, bias, state, lengths, silu, u):
    x, weight = x.astype(np.float64), weight.astype(np.float64)
    B, L, D = x.shape
    K = weight.shape[0]
    before = np.zeros((B, K - 1, D)) if state is None else state.astype(np.float64)
    y, bound, after = np.zeros((B, L, D)), np.zeros((B, L, D)), np.zeros((B, K - 1, D))
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        rows = np.concatenate([before[b], np.where(np.isnan(x[b, :n]), 0, x[b, :n])])
        after[b] = rows[n:]
        v = np.zeros((n, D)) + (0 if bias is None else bias.astype(np.float64))
        size = np.abs(v)
        for k in range(K):
            v = v + weight[k] * rows[k:k + n]
            size = size + np.abs(weight[k] * rows[k:k + n])
        e = (K + 2) * u * size                     # products and additions
        if silu:
            s = v / (1 + np.exp(-v))
            # |d silu / dv| <= 1.1; the exponential: its argument's rounding |v| u and 2 ulp; sum,
            # reciprocal (1 ulp) and product
            e = 1.1 * e + np.abs(s) * (2 * np.abs(v) + 10) * u
            v = s
        y[b, :n], bound[b, :n] = v, e
    return y, after, bound


def state_scan(x, delta, z, A, Bm, Cm, skip, delta_bias, state, lengths, softplus, u, piece=0):
    """`piece`: tokens whose steps a kernel may add up before it takes their common decay."""
    up = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    x, delta, z, A, Bm, Cm, skip, delta_bias = map(up, (x, delta, z, A, Bm, Cm, skip, delta_bias))
    Bn, L, D = x.shape
    N = A.shape[1]
    h = np.zeros((Bn, D, N)) if state is None else up(state).copy()
    size, err = np.abs(h), np.zeros_like(h)       # sum of the terms' magnitudes; what h may be off by
    y, bound = np.zeros((Bn, L, D)), np.zeros((Bn, L, D))
    for b in range(Bn):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        for t in range(n):
            s = delta[b, t] + (0 if delta_bias is None else delta_bias)
            es = 1.0                               # relative error of the step in u: the addition
            if softplus:
                # exponential (argument |v| u, 2 ulp), sum, logarithm, difference, reciprocal, products:
                # at most 12 + 2 |v|; the derivative times v / value is at most 1 + |v|
                es = (1 + np.abs(s)) * es + 12 + 2 * np.abs(s)
                s = np.where(s > 40, s, np.log1p(np.exp(np.minimum(s, 40))))
            es = es * np.ones(D)
            s, es = s[:, None], es[:, None]
            a = np.exp(s * A)
            add = s * Bm[b, t] * x[b, t][:, None]
            # decay: the argument carries the step's error, two roundings and, over a piece, those of
            # the sum of its steps; the exponential 2 ulp; product and sum 2 more
            rel = np.abs(s * A) * (es + 4 + piece) + 6
            err[b] = a * err[b] + u * (a * size[b] * rel + np.abs(add) * (es + 4))
            size[b] = a * size[b] + np.abs(add)
            h[b] = a * h[b] + add
            sums = np.abs(Cm[b, t]) * size[b]
            v = (Cm[b, t] * h[b]).sum(axis=1)
            e = (np.abs(Cm[b, t]) * err[b]).sum(axis=1) + u * (N + 8) * sums.sum(axis=1)
            if skip is not None:
                v = v + skip * x[b, t]
                e = e + 3 * u * (np.abs(skip * x[b, t]) + sums.sum(axis=1))
            if z is not None:
                g = z[b, t] / (1 + np.exp(-z[b, t]))
                e = np.abs(g) * e + np.abs(v * g) * (2 * np.abs(z[b, t]) + 12) * u
                v = v * g
            y[b, t], bound[b, t] = v, e
    return y, h, bound, err + 2 * u * size


def sample_tokens(logits, u, temperature, top_k, top_p, min_p):
    """One row; the word, and how near (relative to the mass) the draw and the cuts came to another one."""
    v = logits.astype(np.float64)
    v = np.where(np.isnan(v), -np.inf, v)
    top = v.max()
    if top == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(np.argmax(v)), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(v == top, 1.0, np.exp((v - top) / temperature))
    w = np.where(np.isnan(w) | (v == -np.inf), 0.0, w)
    order = np.argsort(-v, kind="stable")
    s = w[order]
    n = len(s) if top_k <= 0 else min(top_k, len(s))
    near = 1.0
    if top_p < 1:
        total = s[:n].sum()
        before = np.cumsum(s[:n]) - s[:n]
        gap = np.abs(before - top_p * total) / total
        if len(gap) > 1:
            near = min(near, gap[1:].min())
        n = max(1, int((before < top_p * total).sum()))
    if min_p > 0:
        near = min(near, np.abs(s[:n] - min(min_p, 1.0)).min() if min_p < 1 else 1.0)
        n = max(1, int((s[:n] >= min(min_p, 1.0)).sum()))
    upto = np.cumsum(s[:n])
    u = min(max(u, 0.0), 1.0)
    near = min(near, (np.abs(upto[:-1] - u * upto[-1]) / upto[-1]).min() if n > 1 else 1.0)
    return int(order[min(int((upto <= u * upto[-1]).sum()), n - 1)]), near
