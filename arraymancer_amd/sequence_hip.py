"""Operators of a sequence layer that trains over all tokens at once, for `HipTensor`s: rotary positions, linear attention
with a decay for each head, and group norm with an activation over channels-last tensors.

They stand beside the gated recurrent unit of tensor_hip (src/arraymancer/nn_primitives/nnp_gru.nim:40-500), whose training
walks the tokens one after the other. A layer of them, with the framework's own dense layers around:

    q, k, v   linear(x, Wq) ... reshaped to [batch, tokens, heads, dim]
              q, k = rotary(q, positions, frequencies), rotary(k, positions, frequencies)
              o, state = decay_attention(q, k, v, log_decay, scale=dim ** -0.5)
              y = group_norm(o.reshape(batch * tokens, heads * dim), weight, bias, heads, activation="silu")
              linear(y, Wo)

`decay_attention` takes prompts and training batches, `decay_attention_step` one new token of every sequence; both carry the
same state. Naming and conventions are those of tensor_hip: float32 / float64 tensors, `_into` for a result the caller owns
(rotary alone has one: the others return new tensors, through the C interface they write wherever they are told), `_forward` for
the form that also returns what the backward pass needs, gradients from `_backward` functions. Operands may be strided views; one
whose last dimension has no unit stride is copied on the device first.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _lib
from ._lib import ACT, ROTARY, check
from .metadata import Layout
from .tensor_hip import HipStorage, HipTensor, _same_dtype, toHip, zeros

_INT64 = np.dtype(np.int64)
_FLOAT64 = np.dtype(np.float64)
ROTARY_SCALINGS = ("none", "linear", "base", "parts")


_ENTRIES: dict = {}


def _entry(name: str, t: HipTensor):
    """The entry point of `t`'s element type."""
    fn = _ENTRIES.get((name, t.dtype))
    if fn is None:
        sfx = t.sfx
        if t.dtype.kind != "f":
            raise TypeError(f"{name} is defined for float tensors, not {t.dtype}")
        fn = _ENTRIES[name, t.dtype] = getattr(_lib.load(), f"am_hip_{name}_{sfx}")
    return fn


def _new(shape, dtype) -> HipTensor:
    """`empty` for a shape of ints and a float dtype that have been looked at already: a small operator's call is mostly host time."""
    if len(shape) == 1:
        return HipTensor(Layout(shape, (1,), 0), HipStorage(shape[0], dtype.itemsize), dtype)
    if len(shape) == 2:
        a, b = shape
        return HipTensor(Layout(shape, (b, 1), 0), HipStorage(a * b, dtype.itemsize), dtype)
    if len(shape) == 3:
        a, b, c = shape
        return HipTensor(Layout(shape, (b * c, c, 1), 0), HipStorage(a * b * c, dtype.itemsize), dtype)
    if len(shape) == 4:
        a, b, c, d = shape
        return HipTensor(Layout(shape, (b * c * d, c * d, d, 1), 0), HipStorage(a * b * c * d, dtype.itemsize), dtype)
    strides, n = [], 1
    for d in reversed(shape):
        strides.append(n)
        n *= d
    return HipTensor(Layout(shape, tuple(strides[::-1]), 0), HipStorage(n, dtype.itemsize), dtype)


def _unit_rows(t: HipTensor) -> HipTensor:
    """`t`, or a copy of it, with unit stride in the last dimension."""
    lay = t.layout
    return t if lay.strides[-1] == 1 or lay.shape[-1] == 1 else t.clone()


def _shape(name: str, what: str, t: HipTensor, shape):
    if t.layout.shape != shape:
        raise ValueError(f"{name}: {what} of shape {list(t.shape)}, {list(shape)} expected")


# ---------------------------------------------------------------------- rotary positions
def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, context: int | None = None,
                       fast: float = 32.0, slow: float = 1.0) -> HipTensor:
    """The angles per position of the rot_dim / 2 pairs, base^(-2 i / rot_dim), as the float64 tensor that `rotary` takes.
    For texts `factor` times as long as the trained `context` they are slowed down:
      "linear"  every frequency divided by factor (positions interpolated);
      "base"    a base grown by factor^(rot_dim / (rot_dim - 2)): the fastest pair keeps its frequency, the slowest is divided
                by factor;
      "parts"   pairs that turn more than `fast` times within `context` keep theirs, those that turn less than `slow` times
                are divided by factor, and the shares go linearly between."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rotary_frequencies: {rot_dim} turning elements (an even number is needed)")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}, one of {', '.join(ROTARY_SCALINGS)}")
    if not (base > 0 and factor > 0):
        raise ValueError("rotary_frequencies: base and factor must be positive")
    if scaling == "base":
        if rot_dim < 4:
            raise ValueError('rotary_frequencies: scaling "base" needs two pairs at least')
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = np.power(float(base), -np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "parts":
        if not context or not fast > slow:
            raise ValueError('rotary_frequencies: scaling "parts" needs the trained context and fast > slow')
        turns = context * freq / (2 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        freq = freq * (keep + (1.0 - keep) / factor)
    return toHip(freq)


def _rotate(name, out: HipTensor | None, x: HipTensor, positions: HipTensor | None, frequencies: HipTensor, layout: str, scale: float, inverse: int):
    fn = _entry("rotary", x)
    shape = x.layout.shape
    if len(shape) != 4:
        raise ValueError(f"{name}: a tensor [batch, tokens, heads, dim] is needed, not one of rank {x.rank}")
    B, T, H, D = shape
    if out is not None:
        _same_dtype(x, out)
        _shape(name, "a result", out, x.shape)
        if out.strides[-1] != 1 and D > 1:
            raise ValueError(f"{name}: the last dimension of the result needs unit stride")
    if layout not in ROTARY:
        raise ValueError(f"{name}: unknown layout {layout!r}, one of {', '.join(ROTARY)}")
    if frequencies.dtype != _FLOAT64 or frequencies.rank != 1 or (frequencies.strides[0] != 1 and frequencies.size > 1):
        raise TypeError(f"{name}: frequencies must be a contiguous float64 vector (rotary_frequencies makes one)")
    R = 2 * frequencies.layout.shape[0]
    if R > D:
        raise ValueError(f"{name}: {R} turning elements in a head of {D}")
    pp, pb, pt = None, 0, 0
    if positions is not None:
        if positions.dtype != _INT64:
            raise TypeError(f"{name}: positions must be int64, not {positions.dtype}")
        lay = positions.layout
        if lay.shape == (B, T):
            pb, pt = lay.strides
        elif lay.shape == (T,):
            pt = lay.strides[0]
        else:
            raise ValueError(f"{name}: positions of shape {list(positions.shape)} for {B} sequences of {T} tokens")
        pp = positions.data_ptr()
    if out is None:
        out = _new(shape, x.dtype)
    src = x if x is out else _unit_rows(x)
    xs, os = src.layout.strides, out.layout.strides
    code = fn(B, T, H, D, R, ROTARY[layout], inverse, scale, pp, pb, pt, frequencies.data_ptr(), src.data_ptr(), xs[0], xs[1], xs[2],
              out.data_ptr(), os[0], os[1], os[2])
    if code:
        check(code)
    return out


def rotary(x: HipTensor, positions: HipTensor | None, frequencies: HipTensor, layout: str = "half", scale: float = 1.0) -> HipTensor:
    """x [batch, tokens, heads, dim] with its heads' pairs turned by position * frequency and multiplied by `scale`. The
    first 2 * len(frequencies) elements of a head turn, the rest is copied. layout "half" pairs element i with i + half of
    them, "interleaved" 2 i with 2 i + 1. positions: int64 [batch, tokens] or [tokens], None for 0, 1, 2, ..."""
    return _rotate("rotary", None, x, positions, frequencies, layout, scale, 0)


def rotary_into(out: HipTensor, x: HipTensor, positions: HipTensor | None, frequencies: HipTensor, layout: str = "half",
                scale: float = 1.0) -> HipTensor:
    """`rotary` into a tensor of the caller's; `out` may be `x` (in place), else it must not overlap it."""
    return _rotate("rotary_into", out, x, positions, frequencies, layout, scale, 0)


def rotary_backward(gradient: HipTensor, positions: HipTensor | None, frequencies: HipTensor, layout: str = "half",
                    scale: float = 1.0) -> HipTensor:
    """The gradient of `rotary` with respect to x: the turn back, with the same scale."""
    return _rotate("rotary_backward", None, gradient, positions, frequencies, layout, scale, 1)


# ---------------------------------------------------------------------- linear attention with decay
def _attention_sizes(name, q, k, v, log_decay, lead):
    """Checks q [*lead, heads, dk], k [*lead, kv_heads, dk], v [*lead, kv_heads, dv] and log_decay [heads]."""
    qs, ks, vs = q.layout.shape, k.layout.shape, v.layout.shape
    if not (len(qs) == len(ks) == len(vs) == lead + 2):
        raise ValueError(f"{name}: q, k and v of rank {lead + 2} are needed, not {q.rank}, {k.rank} and {v.rank}")
    dt = q.dtype
    if k.dtype is not dt or v.dtype is not dt or log_decay.dtype is not dt:
        _same_dtype(q, k, v, log_decay)
    front, H, dk = qs[:lead], qs[lead], qs[lead + 1]
    KH, dv = vs[lead:]
    if ks != front + (KH, dk) or vs[:lead] != front:
        raise ValueError(f"{name}: q {list(qs)}, k {list(ks)} and v {list(vs)} do not belong together")
    if H and (KH == 0 or H % KH):
        raise ValueError(f"{name}: {H} heads cannot share {KH} key / value heads evenly")
    _shape(name, "log_decay", log_decay, (H,))
    return front, H, KH, dk, dv


def _head_state(name, t: HipTensor, shape, like: HipTensor):
    """Pointer and (batch, head) strides of a state [batch, heads, dk, dv] whose heads are contiguous."""
    if t.dtype is not like.dtype:
        _same_dtype(like, t)
    _shape(name, "a state", t, shape)
    s = t.layout.strides
    if (s[3] != 1 and shape[3] > 1) or (s[2] != shape[3] and shape[2] > 1):
        raise ValueError(f"{name}: each head of a state must be contiguous")
    return t.data_ptr(), s[0], s[1]


def _lengths(name, lengths: HipTensor | None, batch: int):
    if lengths is None:
        return None
    if lengths.dtype != _INT64:
        raise TypeError(f"{name}: lengths must be int64, not {lengths.dtype}")
    if lengths.shape != (batch,) or not lengths.is_C_contiguous():
        raise ValueError(f"{name}: lengths must be a contiguous vector of {batch} values")
    return lengths.data_ptr()


def _rows(t: HipTensor):
    return (t.data_ptr(),) + t.layout.strides[:-1]


def decay_attention(q: HipTensor, k: HipTensor, v: HipTensor, log_decay: HipTensor, state: HipTensor | None = None,
                    lengths: HipTensor | None = None, scale: float = 1.0):
    """Linear attention with a decay for each head, over whole sequences: per head S <- e^g S + k^T v, out = scale * q S, from
    `state` (None: zeros). Returns (out, the state behind the last token).
    q [batch, tokens, heads, dk], k [batch, tokens, kv_heads, dk], v [batch, tokens, kv_heads, dv], log_decay [heads] (g <= 0),
    states [batch, heads, dk, dv]; head h reads key / value head h // (heads / kv_heads). lengths: int64 [batch], the tokens
    of each sequence; behind them out is 0. `state` is not changed."""
    name = "decay_attention"
    fn = _entry(name, q)
    (B, T), H, KH, dk, dv = _attention_sizes(name, q, k, v, log_decay, 2)
    s0 = _head_state(name, state, (B, H, dk, dv), q) if state is not None else (None, 0, 0)
    n = _lengths(name, lengths, B)
    q, k, v, g = _unit_rows(q), _unit_rows(k), _unit_rows(v), _unit_rows(log_decay)
    out, end = _new((B, T, H, dv), q.dtype), _new((B, H, dk, dv), q.dtype)
    check(fn(B, T, H, KH, dk, dv, scale, g.data_ptr(), n, *_rows(q), *_rows(k), *_rows(v), *s0,
             *_rows(out), *_rows(end)[:3]))
    return out, end


def decay_attention_backward(gradOutput: HipTensor, q: HipTensor, k: HipTensor, v: HipTensor, log_decay: HipTensor,
                             state: HipTensor | None = None, lengths: HipTensor | None = None, scale: float = 1.0,
                             gradState: HipTensor | None = None):
    """(dq, dk, dv, dstate) of `decay_attention` from the gradient of its output and, where it is used further on, that of the
    state it returned (None: zeros). dk and dv of a shared key / value head are sums over the heads that read it; dstate is
    None where no state went in. The decays are constants of the layer and get no gradient."""
    name = "decay_attention_backward"
    fn = _entry(name, q)
    (B, T), H, KH, dk, dv = _attention_sizes(name, q, k, v, log_decay, 2)
    _same_dtype(q, gradOutput)
    _shape(name, "the output's gradient", gradOutput, (B, T, H, dv))
    s0 = _head_state(name, state, (B, H, dk, dv), q) if state is not None else (None, 0, 0)
    gs = _head_state(name, gradState, (B, H, dk, dv), q) if gradState is not None else (None, 0, 0)
    n = _lengths(name, lengths, B)
    q, k, v, do, g = _unit_rows(q), _unit_rows(k), _unit_rows(v), _unit_rows(gradOutput), _unit_rows(log_decay)
    dq, dkey, dval = _new((B, T, H, dk), q.dtype), _new((B, T, KH, dk), q.dtype), _new((B, T, KH, dv), q.dtype)
    dstate = _new((B, H, dk, dv), q.dtype) if state is not None else None
    check(fn(B, T, H, KH, dk, dv, scale, g.data_ptr(), n, *_rows(do), *_rows(q), *_rows(k), *_rows(v),
             *s0, *gs, *_rows(dq), *_rows(dkey), *_rows(dval), *(_rows(dstate)[:3] if dstate is not None else (None, 0, 0))))
    return dq, dkey, dval, dstate


def decay_attention_step(q: HipTensor, k: HipTensor, v: HipTensor, log_decay: HipTensor, state: HipTensor, scale: float = 1.0) -> HipTensor:
    """One new token of every sequence: `state` [batch, heads, dk, dv] is updated in place and the outputs [batch, heads, dv]
    are returned. q [batch, heads, dk], k [batch, kv_heads, dk], v [batch, kv_heads, dv]."""
    name = "decay_attention_step"
    fn = _entry(name, q)
    (B,), H, KH, dk, dv = _attention_sizes(name, q, k, v, log_decay, 1)
    s = _head_state(name, state, (B, H, dk, dv), q)
    q, k, v, g = _unit_rows(q), _unit_rows(k), _unit_rows(v), _unit_rows(log_decay)
    out = _new((B, H, dv), q.dtype)
    qs, ks, vs = q.layout.strides, k.layout.strides, v.layout.strides
    code = fn(B, H, KH, dk, dv, scale, g.data_ptr(), q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
              *s, out.storage.ptr, H * dv, dv)
    if code:
        check(code)
    return out


# ---------------------------------------------------------------------- group norm
def _channels_last(t: HipTensor):
    """(tensor, row stride of the sample, row stride of a position) of t [batch, ..., channels] with the middle dimensions
    walked as one; a copy where the strides do not allow that."""
    s, sh = t.layout.strides, t.layout.shape
    if len(sh) == 2 and s[1] == 1:
        return t, s[0], sh[1]
    if s[-1] == 1 or sh[-1] == 1:
        step, ok = None, True
        for d in range(t.rank - 2, 0, -1):
            if sh[d] == 1:
                continue
            if step is None:
                step, extent = s[d], sh[d]
            else:
                ok = ok and s[d] == step * extent
                extent *= sh[d]
        if ok:
            return t, s[0], step if step is not None else sh[-1]
    t = t.clone()
    return t, t.strides[0], t.shape[-1]


def _norm_sizes(name, x: HipTensor, weight, bias, groups: int, activation: str):
    shape = x.layout.shape
    if len(shape) < 2:
        raise ValueError(f"{name}: a tensor [batch, ..., channels] is needed")
    if activation not in ACT:
        raise ValueError(f"{name}: unknown activation {activation!r}, one of {', '.join(ACT)}")
    C = shape[-1]
    spatial = 1
    for d in shape[1:-1]:
        spatial *= d
    if groups < 1 or C % groups:
        raise ValueError(f"{name}: {C} channels cannot form {groups} groups")
    for what, w in (("weight", weight), ("bias", bias)):
        if w is not None:
            if w.dtype is not x.dtype:
                _same_dtype(x, w)
            ws = w.layout.shape
            if ws != (C,) and ws != (1, C):
                raise ValueError(f"{name}: {what} of shape {list(w.shape)} for {C} channels")
    return shape[0], spatial, C


def _vector(t: HipTensor | None):
    """`t` [channels] or [1, channels] with its channels next to each other."""
    return t if t is None else _unit_rows(t)


def _ptr(t: HipTensor | None):
    return None if t is None else t.data_ptr()


def _normalise(name, x, weight, bias, groups, eps, activation, keep):
    fn = _entry("group_norm", x)
    B, S, C = _norm_sizes(name, x, weight, bias, groups, activation)
    src, sn, ss = _channels_last(x)
    w, b = _vector(weight), _vector(bias)
    y = _new(x.layout.shape, x.dtype)
    mean = rstd = None
    if keep:
        make = _new if S * C else zeros
        mean, rstd = make((B, groups), x.dtype), make((B, groups), x.dtype)
    code = fn(B, S, C, groups, eps, ACT[activation], src.data_ptr(), sn, ss, _ptr(w), _ptr(b), y.storage.ptr, S * C, C, _ptr(mean), _ptr(rstd))
    if code:
        check(code)
    return y, mean, rstd


def group_norm(x: HipTensor, weight: HipTensor | None, bias: HipTensor | None, groups: int, eps: float = 1e-5,
               activation: str = "none") -> HipTensor:
    """act((x - mean) / sqrt(variance + eps) * weight + bias) of a channels-last tensor [batch, ..., channels], mean and
    variance over each sample's positions and the channels / groups neighbouring channels of a group. weight and bias
    ([channels] or [1, channels]) may be None. activation: "none", "relu", "silu". A tensor whose channels are not next to
    each other in memory (an image [batch, channels, height, width] permuted) is copied first."""
    return _normalise("group_norm", x, weight, bias, groups, eps, activation, False)[0]


def group_norm_forward(x: HipTensor, weight: HipTensor | None, bias: HipTensor | None, groups: int, eps: float = 1e-5,
                       activation: str = "none"):
    """`group_norm`, keeping what the backward pass needs: (y, mean, 1 / deviation), the latter [batch, groups]."""
    return _normalise("group_norm_forward", x, weight, bias, groups, eps, activation, True)


def group_norm_backward(gradOutput: HipTensor, x: HipTensor, weight: HipTensor | None, bias: HipTensor | None, mean: HipTensor,
                        rstd: HipTensor, groups: int, activation: str = "none"):
    """(dx, dweight, dbias) from the gradient of the output, the inputs of `group_norm_forward` and the mean and rstd that it
    returned; dweight and dbias have the shapes of weight and bias and are None where those are."""
    name = "group_norm_backward"
    fn = _entry(name, x)
    B, S, C = _norm_sizes(name, x, weight, bias, groups, activation)
    dt = x.dtype
    if gradOutput.dtype is not dt or mean.dtype is not dt or rstd.dtype is not dt:
        _same_dtype(x, gradOutput, mean, rstd)
    _shape(name, "the output's gradient", gradOutput, x.layout.shape)
    _shape(name, "mean", mean, (B, groups))
    _shape(name, "rstd", rstd, (B, groups))
    src, xn, xs = _channels_last(x)
    dy, gn, gs = _channels_last(gradOutput)
    w, b = _vector(weight), _vector(bias)
    m, r = (t if t.layout.strides == (groups, 1) else t.asContiguous() for t in (mean, rstd))
    dx = _new(x.layout.shape, dt)
    dw = _new(weight.layout.shape, dt) if weight is not None else None
    db = _new(bias.layout.shape, dt) if bias is not None else None
    code = fn(B, S, C, groups, ACT[activation], dy.data_ptr(), gn, gs, src.data_ptr(), xn, xs, _ptr(w), _ptr(b), m.data_ptr(), r.data_ptr(),
              dx.storage.ptr, S * C, C, _ptr(dw), _ptr(db))
    if code:
        check(code)
    return dx, dw, db
