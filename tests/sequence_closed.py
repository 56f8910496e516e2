"""Linear attention with decay in its closed form (no recurrence), in float64 NumPy and over all heads at once: what the larger
sizes of tests/test_sequence_paths_gpu.py are compared with. Arguments and results as in tests/sequence_reference.py; fed with
absolute values it gives the sums of the absolute terms."""
import numpy as np

from sequence_reference import shared


def _parts(q, k, v, g, lengths):
    B, T, H, _ = q.shape
    n = np.full(B, T) if lengths is None else np.clip(lengths, 0, T)
    live = (np.arange(T)[None] < n[:, None])[:, None, :, None]
    front = lambda x: np.where(live, x.astype(np.float64).transpose(0, 2, 1, 3), 0.0)       # [batch, heads, tokens, dim]
    g = g.astype(np.float64)
    at = np.arange(T)
    apart = at[:, None] - at[None, :]
    power = lambda e: np.where(e == 0, 1.0, np.exp(g[(...,) + (None,) * e.ndim] * np.maximum(e, 1)))
    mask = np.where(apart >= 0, power(np.maximum(apart, 0)), 0.0)                           # e^(g (i - j)), [heads, i, j]
    reach = power(at + 1)[None, :, :, None]                                                 # e^(g (i + 1))
    left = np.stack([power(np.maximum(m - 1 - at, 0)) for m in n])[..., None]               # e^(g (n - 1 - j))
    whole = np.stack([power(np.array(m)) for m in n])[..., None, None]                      # e^(g n)
    return front(q), front(shared(k, H)), front(shared(v, H)), front, mask, reach, left, whole


def attention(q, k, v, g, state=None, lengths=None, scale=1.0):
    Q, K, V, _, mask, reach, left, whole = _parts(q, k, v, g, lengths)
    out = (Q @ K.transpose(0, 1, 3, 2) * mask) @ V
    end = (K * left).transpose(0, 1, 3, 2) @ V
    if state is not None:
        S = state.astype(np.float64)
        out = out + reach * (Q @ S)
        end = end + whole * S
    return scale * out.transpose(0, 2, 1, 3), end


def attention_backward(go, q, k, v, g, state=None, lengths=None, scale=1.0, gs=None):
    Q, K, V, front, mask, reach, left, whole = _parts(q, k, v, g, lengths)
    B, H, T, dk = Q.shape
    dO = front(go)
    A, dA = Q @ K.transpose(0, 1, 3, 2) * mask, dO @ V.transpose(0, 1, 3, 2) * mask
    dq, dkey, dval = scale * (dA @ K), scale * (dA.transpose(0, 1, 3, 2) @ Q), scale * (A.transpose(0, 1, 3, 2) @ dO)
    dstate = scale * ((Q * reach).transpose(0, 1, 3, 2) @ dO)
    if state is not None:
        dq = dq + scale * reach * (dO @ state.astype(np.float64).transpose(0, 1, 3, 2))
    if gs is not None:
        G = gs.astype(np.float64)
        dkey, dval, dstate = dkey + left * (V @ G.transpose(0, 1, 3, 2)), dval + left * (K @ G), dstate + whole * G
    back = lambda x: x.transpose(0, 2, 1, 3)
    fold = lambda x: back(x).reshape(B, T, k.shape[2], -1, x.shape[-1]).sum(3)
    return back(dq), fold(dkey), fold(dval), dstate
