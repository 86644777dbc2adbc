"""Operators of recurrent sequence models on Arrays: what the blocks of a model need beside its products
and element-wise statements, for whole prompts and for single tokens, and the draw of the next token.

Upstream has no counterpart: its one model is the LSTM forward written in array statements
(examples/lstm_forward.py:29-49 upstream). Each function records one call that runs in program order; the
mathematics and the kernels' limits stand at cnh_rms_norm, cnh_short_convolution, cnh_state_scan and
cnh_sample_tokens in include/cnhip.h. float32 and float64: operands that are only read are converted to
np.result_type of x and the others where their types differ (integers count as float64); arrays that are
updated in place keep their type and must already have that one. Slices with unit steps are read where
they are, other slices are copied first.
"""
from __future__ import annotations

import numpy as np

from . import _lib as L
from . import lazy
from .array import Array, ArrayView, _ArrayLike, _coerce_scalar, _converted, _is_scalar_like, _is_whole, asarray

_I32, _F64 = np.dtype("int32"), np.dtype("float64")


def _operand(x, what):
    if x is None:
        return None
    if _is_scalar_like(x):
        raise TypeError(f"{what} must be an array, not a scalar")
    return asarray(x)


def _common_type(operands):
    dt = np.result_type(*[o.dtype for o in operands if o is not None])
    return _F64 if dt.kind != "f" else dt


def _as_type(x, dtype):
    return x if x is None or x.dtype == dtype else _converted(x, dtype)


def _updated(x, what, shape, dtype):
    """An array that the call updates in place: a whole one of the right extents and type."""
    if x is None:
        return None
    if not isinstance(x, _ArrayLike):
        raise TypeError(f"{what} is updated in place and must be a charmnumeric Array")
    if not _is_whole(x._region(), x._base().shape):
        raise ValueError(f"{what} is updated in place and must be a whole array, not a slice")
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {x.shape}, expected {tuple(shape)}")
    if x.dtype != dtype:
        raise TypeError(f"{what} is {x.dtype.name}, the call computes in {dtype.name}")
    x._base()._all_ones = False
    return x._base()


def _distinct(updated, read):
    """What a call updates must not be among what it reads."""
    if updated is not None:
        for what, x in read.items():
            if x is not None and x.name == updated.name:
                raise ValueError(f"{what} is a part of the array that the call updates in place")


def _whole(x, what, shape, dtype):
    """An operand that is read as a whole (slices are copied out first)."""
    if x is None:
        return None
    if tuple(x.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {x.shape}, expected {tuple(shape)}")
    x = _as_type(x, dtype)
    return x.copy() if isinstance(x, ArrayView) and not _is_whole(x.region, x.base.shape) else x


def _counts(x, what, n):
    """Integers, one per sequence or row: held to 32 bits, here where they are the host's, by the executor
    where they are an Array of 64 bits."""
    if not isinstance(x, _ArrayLike):
        x = np.asarray(x)
        if x.dtype.kind in "iu":
            here, to = np.iinfo(x.dtype), np.iinfo(_I32)
            x = np.clip(x, max(here.min, to.min), min(here.max, to.max))
        elif x.dtype.kind != "b":
            raise TypeError(f"{what} must be integers, got {x.dtype.name}")
        x = asarray(x.astype(_I32))
    if x.dtype.kind != "i":
        raise TypeError(f"{what} must be integers, got {x.dtype.name}")
    return _whole(x, what, (n,), x.dtype)


def _lengths(x, batch):
    return None if x is None else _counts(x, "lengths", batch)


def _sliced(x, even_rows=False):
    """x itself where a kernel can read it in place: whole, or a slice with unit steps (and, where the
    kernel walks all rows at one distance, a rank-3 slice that leaves out no row)."""
    if not isinstance(x, ArrayView) or _is_whole(x.region, x.base.shape):
        return x
    if any(st != 1 for st in x.region[2]):
        return x.copy()
    if even_rows and x.ndims == 3 and x.shape[0] > 1 and x.shape[1] != x.base.shape[1]:
        return x.copy()
    return x


def _name(x):
    return 0 if x is None else x.name


def _ref(x):
    o = L.Operand()
    o.region.is_global = 1
    if x is not None:
        o.name = x.name
        region = x._region()
        if region is not None and not _is_whole(region, x._base().shape):
            o.region = L.Region.make(*region)
    return o


def _record(kind, out, args):
    lazy.record_call(lazy.Call(out.name, kind, out.wire_dtype(), args))
    return out


def _rows_of(x, what, call):
    if x.ndims not in (2, 3):
        raise ValueError(f"{call}: {what} must be (batch, length, n) or (batch, n), got rank {x.ndims}")
    return tuple(x.shape[:-1])


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """Root-mean-square norm along the last dimension: x / sqrt(mean(x**2) + eps) * weight, weight of the
    last dimension's length (None: ones). With `residual`, an Array of x's shape, r = x + residual is
    normalised instead and residual becomes r: the residual stream of a block, updated on the way."""
    x, weight = _operand(x, "x"), _operand(weight, "weight")
    eps = float(eps)
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    dtype = _common_type([x, weight])
    if isinstance(residual, _ArrayLike) and residual.dtype.kind == "f":
        dtype = np.result_type(dtype, residual.dtype)
    residual = _updated(residual, "residual", x.shape, dtype)
    _distinct(residual, {"x": x, "weight": weight})
    weight = _whole(weight, "weight", x.shape[-1:], dtype)
    x = _sliced(_as_type(x, dtype), even_rows=True)
    out = Array(x.shape, dtype)
    return _record("rms_norm", out, L.XRmsNorm(_ref(x), _name(residual), _name(weight), out.name, eps))


def short_convolution(x, weight, bias=None, state=None, lengths=None, activation="silu"):
    """Causal convolution of every channel along its tokens. x: (batch, length, channels), or (batch,
    channels) for one token of each sequence; weight: (taps, channels), 1 to 8 taps, the last one for the
    token itself; bias: (channels,). activation: "silu" or None.

    state, (batch, taps - 1, channels): the rows in front of the first token (None: zeros), which become
    the last rows of each sequence, so that the next call goes on where this one ended. lengths: how many
    of the `length` tokens each sequence has, integers of any width (None: all); rows of the result behind
    them are zeros."""
    x, weight, bias = _operand(x, "x"), _operand(weight, "weight"), _operand(bias, "bias")
    lead = _rows_of(x, "x", "short_convolution")
    if activation not in ("silu", None):
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    if weight is None or weight.ndims != 2 or not 1 <= weight.shape[0] <= 8:
        raise ValueError("weight must be (taps, channels) with 1 to 8 taps")
    channels, taps = x.shape[-1], weight.shape[0]
    if taps == 1 and state is not None:
        raise ValueError("a convolution of one tap has no state")
    dtype = _common_type([x, weight, bias])
    if isinstance(state, _ArrayLike) and state.dtype.kind == "f":
        dtype = np.result_type(dtype, state.dtype)
    state = _updated(state, "state", (lead[0], taps - 1, channels), dtype)
    _distinct(state, {"x": x, "weight": weight, "bias": bias})
    weight, bias = _whole(weight, "weight", (taps, channels), dtype), _whole(bias, "bias", (channels,), dtype)
    lengths = _lengths(lengths, lead[0])
    x = _sliced(_as_type(x, dtype))
    out = Array(x.shape, dtype)
    return _record("short_convolution", out, L.XShortConvolution(
        _ref(x), _name(weight), _name(bias), _name(state), _name(lengths), out.name, 1 if activation else 0))


def state_scan(x, delta, A, B, C, skip=None, z=None, delta_bias=None, state=None, lengths=None, softplus=True):
    """Selective state space scan: per channel, with s = softplus(delta + delta_bias),
        h = exp(s * A) * h + s * B * x,   y = (sum over states of C * h + skip * x) * z * sigmoid(z)
    from token to token. x, delta, z: (batch, length, channels), or (batch, channels) for one token of each
    sequence; B, C: (batch, length, states) or (batch, states), 1 to 256 states; A: (channels, states);
    skip, delta_bias: (channels,). None stands for no gate (z), no skip, no bias; softplus=False takes
    delta + delta_bias as it is.

    state, (batch, channels, states): h in front of the first token (None: zeros), which becomes h behind
    the last one. lengths as for short_convolution."""
    x, delta, A, B, C = (_operand(v, n) for v, n in ((x, "x"), (delta, "delta"), (A, "A"), (B, "B"), (C, "C")))
    skip, z, delta_bias = _operand(skip, "skip"), _operand(z, "z"), _operand(delta_bias, "delta_bias")
    lead, channels = _rows_of(x, "x", "state_scan"), x.shape[-1]
    if A is None or A.ndims != 2 or A.shape[0] != channels or not 1 <= A.shape[1] <= 256:
        raise ValueError(f"A must be ({channels}, states) with 1 to 256 states")
    states = A.shape[1]
    for v, what, last in ((delta, "delta", channels), (z, "z", channels), (B, "B", states), (C, "C", states)):
        if (v is None and what != "z") or (v is not None and tuple(v.shape) != lead + (last,)):
            raise ValueError(f"{what} must have shape {lead + (last,)}, got {None if v is None else v.shape}")
    dtype = _common_type([x, delta, A, B, C, skip, z, delta_bias])
    if isinstance(state, _ArrayLike) and state.dtype.kind == "f":
        dtype = np.result_type(dtype, state.dtype)
    state = _updated(state, "state", (lead[0], channels, states), dtype)
    _distinct(state, dict(x=x, delta=delta, A=A, B=B, C=C, skip=skip, z=z, delta_bias=delta_bias))
    A = _whole(A, "A", A.shape, dtype)
    skip, delta_bias = (_whole(v, n, (channels,), dtype) for v, n in ((skip, "skip"), (delta_bias, "delta_bias")))
    lengths = _lengths(lengths, lead[0])
    x, delta, z, B, C = (_sliced(_as_type(v, dtype)) if v is not None else None for v in (x, delta, z, B, C))
    out = Array(x.shape, dtype)
    return _record("state_scan", out, L.XStateScan(
        _ref(x), _ref(delta), _ref(z), _ref(B), _ref(C), _name(A), _name(skip), _name(delta_bias), _name(state),
        _name(lengths), out.name, 1 if softplus else 0))


def _setting(v, what, rows, dtype, lowest, highest):
    """(scalar, array or None) of a setting that is either one number or one per row."""
    if not _is_scalar_like(v):
        return 0, _counts(v, what, rows) if dtype == _I32 else _whole(_operand(v, what), what, (rows,), dtype)
    v = _coerce_scalar(v)
    if dtype == _I32 and not isinstance(v, int):
        raise TypeError(f"{what} must be an integer, got {v!r}")
    if not lowest <= v <= highest:
        raise ValueError(f"{what} must lie between {lowest} and {highest}, got {v}")
    return v, None


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One index per row of logits (rows, vocab) or (vocab,), drawn with the random numbers u (rows,) of
    [0, 1), for instance random.uniform((rows,), seed): an int32 Array (rows,).

    Weights are exp((logit - largest) / temperature); top_k > 0 keeps the k largest (ties: the lowest
    indices), top_p < 1 the shortest run of those, in descending order, whose mass reaches top_p of theirs,
    min_p > 0 those of at least min_p times the largest weight. The index drawn is the first in descending order
    at which the running mass exceeds u times the mass kept. temperature 0 takes the largest logit. -inf
    and NaN are never drawn; a row that holds nothing else gives -1. Every setting may be an array with one
    entry per row."""
    logits, u = _operand(logits, "logits"), _operand(u, "u")
    if logits.ndims > 2:
        raise ValueError(f"logits must be (rows, vocab) or (vocab,), got rank {logits.ndims}")
    rows = logits.shape[0] if logits.ndims == 2 else 1
    if logits.shape[-1] > 1 << 22:
        raise NotImplementedError("vocabularies beyond 2**22 words are not supported")
    if u is None:
        raise ValueError("sample_tokens needs random numbers")
    u = _whole(u, "u", (rows,), _F64)
    inf = float("inf")
    t, ts = _setting(temperature, "temperature", rows, _F64, 0, inf)
    k, ks = _setting(top_k, "top_k", rows, _I32, 0, (1 << 31) - 1)
    p, ps = _setting(top_p, "top_p", rows, _F64, 0, inf)
    m, ms = _setting(min_p, "min_p", rows, _F64, 0, 1)
    logits = _sliced(_as_type(logits, _common_type([logits])))
    out = Array((rows,), _I32)
    return _record("sample_tokens", out, L.XSampleTokens(
        _ref(logits), _name(u), _name(ts), _name(ks), _name(ps), _name(ms), out.name, k, t, p, m))
