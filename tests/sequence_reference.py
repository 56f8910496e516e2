"""The sequence operators from their definitions, in float64 NumPy: what tests/test_sequence_gpu.py compares with. Each
function also serves for bounds: fed with absolute values it gives the sum of the absolute terms of a result, and a result
whose terms pass through n roundings each is off by at most n half steps of that sum."""
import numpy as np


def rotary(x, positions, freq, layout="half", scale=1.0, inverse=False):
    x = x.astype(np.float64)
    n = len(freq)
    angle = positions.astype(np.float64)[..., None] * freq          # [batch, tokens, pairs]
    if inverse:
        angle = -angle
    c, s = np.cos(angle)[:, :, None] * scale, np.sin(angle)[:, :, None] * scale
    out = x.copy()
    first, second = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., first], x[..., second]
    out[..., first] = a * c - b * s
    out[..., second] = b * c + a * s
    return out


def shared(x, heads):
    """Every head's own copy of the key / value head it reads."""
    return np.repeat(x, heads // x.shape[-2], axis=-2)


def attention(q, k, v, g, state=None, lengths=None, scale=1.0):
    """The recurrence: (out, last state)."""
    q, g = q.astype(np.float64), g.astype(np.float64)
    B, T, H, dk = q.shape
    k, v = shared(k.astype(np.float64), H), shared(v.astype(np.float64), H)
    S = np.zeros((B, H, dk, v.shape[-1])) if state is None else state.astype(np.float64).copy()
    out = np.zeros((B, T, H, v.shape[-1]))
    lam = np.exp(g)[:, None, None]
    for b in range(B):
        for t in range(T if lengths is None else min(max(int(lengths[b]), 0), T)):
            S[b] = S[b] * lam + k[b, t][:, :, None] * v[b, t][:, None, :]
            out[b, t] = scale * np.einsum("hi,hij->hj", q[b, t], S[b])
    return out, S


def attention_backward(go, q, k, v, g, state=None, lengths=None, scale=1.0, gs=None):
    """(dq, dk, dv, dstate): the recurrence differentiated step by step."""
    q, g, go = q.astype(np.float64), g.astype(np.float64), go.astype(np.float64)
    B, T, H, dk = q.shape
    KH, dv = v.shape[-2:]
    kk, vv = shared(k.astype(np.float64), H), shared(v.astype(np.float64), H)
    lam = np.exp(g)[:, None, None]
    dq, dkey, dval = np.zeros((B, T, H, dk)), np.zeros((B, T, H, dk)), np.zeros((B, T, H, dv))
    dS0 = np.zeros((B, H, dk, dv))
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        S = np.zeros((H, dk, dv)) if state is None else state[b].astype(np.float64)
        for t in range(n):
            S = S * lam + kk[b, t][:, :, None] * vv[b, t][:, None, :]
            dq[b, t] = scale * np.einsum("hj,hij->hi", go[b, t], S)
        R = np.zeros((H, dk, dv)) if gs is None else gs[b].astype(np.float64)
        for t in reversed(range(n)):
            R = R + scale * q[b, t][:, :, None] * go[b, t][:, None, :]
            dkey[b, t] = np.einsum("hj,hij->hi", vv[b, t], R)
            dval[b, t] = np.einsum("hi,hij->hj", kk[b, t], R)
            R = R * lam
        dS0[b] = R
    fold = lambda x: x.reshape(B, T, KH, H // KH, x.shape[-1]).sum(3)
    return dq, fold(dkey), fold(dval), dS0


def _act(z, activation):
    if activation == "relu":
        return np.where(z > 0, z, 0.0)
    if activation == "silu":
        return z / (1 + np.exp(-z))
    return z


def _slope(z, activation):
    if activation == "relu":
        return (z > 0).astype(np.float64)
    if activation == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def _grouped(x, groups):
    return x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)


def norm_stats(x, groups, eps):
    v = _grouped(x.astype(np.float64), groups)
    mean = v.mean((1, 3), keepdims=True)
    return mean, 1 / np.sqrt(((v - mean) ** 2).mean((1, 3), keepdims=True) + eps)


def norm(x, w, b, groups, eps, activation="none"):
    mean, rstd = norm_stats(x, groups, eps)
    z = ((_grouped(x.astype(np.float64), groups) - mean) * rstd).reshape(x.shape)
    if w is not None:
        z = z * w.astype(np.float64)
    if b is not None:
        z = z + b.astype(np.float64)
    return _act(z, activation)


def norm_backward(dy, x, w, b, groups, eps, activation="none"):
    """(dx, dweight, dbias)."""
    C = x.shape[-1]
    mean, rstd = norm_stats(x, groups, eps)
    xhat = ((_grouped(x.astype(np.float64), groups) - mean) * rstd).reshape(x.shape)
    w64 = np.ones(C) if w is None else w.astype(np.float64).reshape(-1)
    z = xhat * w64 + (0.0 if b is None else b.astype(np.float64).reshape(-1))
    dz = dy.astype(np.float64) * _slope(z, activation)
    d, h = _grouped(dz * w64, groups), _grouped(xhat, groups)
    dx = rstd * (d - d.mean((1, 3), keepdims=True) - h * (d * h).mean((1, 3), keepdims=True))
    flat = lambda a: a.reshape(-1, C)
    return dx.reshape(x.shape), flat(dz * xhat).sum(0), flat(dz).sum(0)
