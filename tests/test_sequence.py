"""The sequence operators without a device: what they refuse (before anything reaches the GPU), the frequencies, and the
definitions that the device tests compare with, checked against differences."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import arraymancer_amd as am
import sequence_reference as ref
from arraymancer_amd import _lib, metadata as md
from arraymancer_amd.tensor_hip import HipTensor


class _Nowhere:
    ptr, nelems, itemsize = 0x1000, 1 << 20, 4


def fake(*shape, dtype=np.float32):
    return HipTensor(md.contiguous(shape), _Nowhere(), dtype)


P = ctypes.c_void_p(0x1000)


def rotary_args(**kw):
    a = dict(batch=2, tokens=3, heads=4, dim=8, rot=8, layout=0, inverse=0, scale=1.0, pos=None, pb=0, pt=0, freq=P, x=P, xb=96, xt=32, xh=8,
             out=P, ob=96, ot=32, oh=8)
    a.update(kw)
    return list(a.values())


def attention_args(**kw):
    a = dict(batch=2, tokens=3, heads=4, kv=2, dk=8, dv=8, scale=1.0, g=P, lengths=None, q=P, qb=96, qt=32, qh=8, k=P, kb=48, kt=16, kh=8,
             v=P, vb=48, vt=16, vh=8, s0=None, s0b=0, s0h=0, out=P, ob=96, ot=32, oh=8, s1=P, s1b=256, s1h=64)
    a.update(kw)
    return list(a.values())


def backward_args(**kw):
    a = dict(batch=2, tokens=3, heads=4, kv=2, dk=8, dv=8, scale=1.0, g=P, lengths=None, go=P, gb=96, gt=32, gh=8, q=P, qb=96, qt=32, qh=8,
             k=P, kb=48, kt=16, kh=8, v=P, vb=48, vt=16, vh=8, s0=None, s0b=0, s0h=0, gs=None, gsb=0, gsh=0, dq=P, dqb=96, dqt=32, dqh=8,
             dk_=P, dkb=48, dkt=16, dkh=8, dv_=P, dvb=48, dvt=16, dvh=8, gs0=None, gs0b=0, gs0h=0)
    a.update(kw)
    return list(a.values())


def step_args(**kw):
    a = dict(batch=2, heads=4, kv=2, dk=8, dv=8, scale=1.0, g=P, q=P, qb=32, qh=8, k=P, kb=16, kh=8, v=P, vb=16, vh=8, s=P, sb=256, sh=64,
             out=P, ob=32, oh=8)
    a.update(kw)
    return list(a.values())


def norm_args(**kw):
    a = dict(batch=2, spatial=3, channels=8, groups=2, eps=1e-5, act=0, x=P, xn=24, xs=8, w=None, b=None, y=P, yn=24, ys=8, mean=None, rstd=None)
    a.update(kw)
    return list(a.values())


def norm_backward_args(**kw):
    a = dict(batch=2, spatial=3, channels=8, groups=2, act=0, dy=P, dyn=24, dys=8, x=P, xn=24, xs=8, w=None, b=None, mean=P, rstd=P, dx=P, dxn=24,
             dxs=8, dw=None, db=None)
    a.update(kw)
    return list(a.values())


REFUSED = [
    ("rotary", rotary_args, dict(layout=2), "layout"), ("rotary", rotary_args, dict(rot=7), "turning"), ("rotary", rotary_args, dict(rot=10), "turning"),
    ("rotary", rotary_args, dict(tokens=-1), "negative"), ("rotary", rotary_args, dict(x=None), "null"), ("rotary", rotary_args, dict(freq=None), "null"),
    ("rotary", rotary_args, dict(oh=0), "broadcast"), ("rotary", rotary_args, dict(ot=0), "broadcast"), ("rotary", rotary_args, dict(dim=1 << 24, rot=8), "large"),
    ("decay_attention", attention_args, dict(dk=0), "elements"), ("decay_attention", attention_args, dict(dv=257), "elements"),
    ("decay_attention", attention_args, dict(kv=3), "share"), ("decay_attention", attention_args, dict(kv=0), "share"),
    ("decay_attention", attention_args, dict(batch=-1), "negative"), ("decay_attention", attention_args, dict(g=None), "null"),
    ("decay_attention", attention_args, dict(v=None), "null"), ("decay_attention", attention_args, dict(out=None), "null"),
    ("decay_attention", attention_args, dict(ot=0), "broadcast"), ("decay_attention", attention_args, dict(s1h=0), "broadcast"),
    ("decay_attention_backward", backward_args, dict(dv=300), "elements"), ("decay_attention_backward", backward_args, dict(kv=3), "share"),
    ("decay_attention_backward", backward_args, dict(dq=None), "null"), ("decay_attention_backward", backward_args, dict(go=None), "null"),
    ("decay_attention_backward", backward_args, dict(dkt=0), "broadcast"), ("decay_attention_backward", backward_args, dict(gs0=P), "broadcast"),
    ("decay_attention_step", step_args, dict(dk=257), "elements"), ("decay_attention_step", step_args, dict(kv=8), "share"),
    ("decay_attention_step", step_args, dict(s=None), "null"), ("decay_attention_step", step_args, dict(sb=0), "broadcast"),
    ("group_norm", norm_args, dict(groups=3), "groups"), ("group_norm", norm_args, dict(groups=0), "groups"), ("group_norm", norm_args, dict(act=3), "activation"),
    ("group_norm", norm_args, dict(eps=-1.0), "eps"), ("group_norm", norm_args, dict(eps=float("nan")), "eps"), ("group_norm", norm_args, dict(mean=P), "together"),
    ("group_norm", norm_args, dict(spatial=-1), "negative"), ("group_norm", norm_args, dict(y=None), "null"), ("group_norm", norm_args, dict(ys=0), "broadcast"),
    ("group_norm_backward", norm_backward_args, dict(act=-1), "activation"), ("group_norm_backward", norm_backward_args, dict(mean=None), "null"),
    ("group_norm_backward", norm_backward_args, dict(dxn=0), "broadcast"), ("group_norm_backward", norm_backward_args, dict(groups=5), "groups"),
]


@pytest.mark.parametrize("sfx", ["f32", "f64"])
@pytest.mark.parametrize("entry,args,change,word", REFUSED, ids=lambda v: str(v) if not callable(v) else "")
def test_the_c_entry_points_refuse(entry, args, change, word, sfx):
    L = am.load_library()
    assert getattr(L, f"am_hip_{entry}_{sfx}")(*args(**change)) in (_lib.AM_E_ARG, _lib.AM_E_SHAPE)
    assert word in _lib.last_error() and f"am_hip_{entry}_{sfx}" in _lib.last_error()


@pytest.mark.parametrize("entry,args,change", [("rotary", rotary_args, dict(batch=0)), ("rotary", rotary_args, dict(heads=0, x=None, out=None)),
                                               ("decay_attention", attention_args, dict(batch=0)), ("decay_attention", attention_args, dict(heads=0, kv=0)),
                                               ("decay_attention_step", step_args, dict(batch=0)), ("group_norm", norm_args, dict(batch=0)),
                                               ("group_norm_backward", norm_backward_args, dict(channels=0))])
def test_nothing_to_do_needs_no_device(entry, args, change):
    assert getattr(am.load_library(), f"am_hip_{entry}_f32")(*args(**change)) == _lib.AM_OK


def test_the_python_layer_refuses():
    x, f = fake(2, 3, 4, 8), fake(4, dtype=np.float64)
    pos = fake(2, 3, dtype=np.int64)
    into = lambda **kw: am.rotary_into(**{**dict(out=x, x=x, positions=pos, frequencies=f), **kw})
    for kw, err in ((dict(x=fake(3, 4, 8)), ValueError), (dict(frequencies=fake(4)), TypeError), (dict(frequencies=fake(5, dtype=np.float64)), ValueError),
                    (dict(positions=fake(2, 3, dtype=np.int32)), TypeError), (dict(positions=fake(3, 2, dtype=np.int64)), ValueError),
                    (dict(layout="pairs"), ValueError), (dict(out=fake(2, 3, 4, 9)), ValueError), (dict(out=fake(2, 3, 8, 4).permute(0, 1, 3, 2)), ValueError),
                    (dict(x=fake(2, 3, 4, 8, dtype=np.float64)), TypeError), (dict(x=fake(2, 3, 4, 8, dtype=np.int32)), TypeError)):
        with pytest.raises(err):
            into(**kw)
    q, k, v, g, s = fake(2, 3, 4, 8), fake(2, 3, 2, 8), fake(2, 3, 2, 6), fake(4), fake(2, 4, 8, 6)
    for kw, err in ((dict(q=fake(2, 4, 8)), ValueError), (dict(k=fake(2, 3, 2, 9)), ValueError), (dict(k=fake(2, 3, 3, 8), v=fake(2, 3, 3, 6)), ValueError),
                    (dict(v=fake(2, 2, 2, 6)), ValueError), (dict(log_decay=fake(3)), ValueError), (dict(log_decay=fake(4, dtype=np.float64)), TypeError),
                    (dict(state=fake(2, 4, 6, 8)), ValueError), (dict(state=fake(2, 4, 6, 8).permute(0, 1, 3, 2)), ValueError),
                    (dict(lengths=fake(2, dtype=np.int32)), TypeError), (dict(lengths=fake(3, dtype=np.int64)), ValueError),
                    (dict(q=fake(2, 3, 4, 8, dtype=np.int64)), TypeError)):
        with pytest.raises(err):
            am.decay_attention(**{**dict(q=q, k=k, v=v, log_decay=g), **kw})
        with pytest.raises(err):
            am.decay_attention_backward(**{**dict(gradOutput=fake(2, 3, 4, 6), q=q, k=k, v=v, log_decay=g), **kw})
    with pytest.raises(ValueError):
        am.decay_attention_backward(fake(2, 3, 4, 8), q, k, v, g)
    with pytest.raises(ValueError):
        am.decay_attention_backward(fake(2, 3, 4, 6), q, k, v, g, gradState=fake(2, 4, 8, 8))
    with pytest.raises(ValueError):
        am.decay_attention_step(q, k, v, g, s)
    with pytest.raises(ValueError):
        am.decay_attention_step(fake(2, 4, 8), fake(2, 2, 8), fake(2, 2, 6), g, fake(2, 4, 6, 8))
    n = fake(2, 5, 8)
    for kw, err in ((dict(x=fake(8)), ValueError), (dict(groups=3), ValueError), (dict(groups=0), ValueError), (dict(activation="gelu"), ValueError),
                    (dict(weight=fake(4)), ValueError), (dict(bias=fake(8, 1)), ValueError), (dict(weight=fake(8, dtype=np.float64)), TypeError),
                    (dict(x=fake(2, 8, dtype=np.int32)), TypeError)):
        with pytest.raises(err):
            am.group_norm(**{**dict(x=n, weight=fake(8), bias=fake(8), groups=2), **kw})
    for kw, err in ((dict(gradOutput=fake(2, 8)), ValueError), (dict(mean=fake(2, 4)), ValueError), (dict(rstd=fake(1, 2)), ValueError),
                    (dict(mean=fake(2, 2, dtype=np.float64)), TypeError)):
        with pytest.raises(err):
            am.group_norm_backward(**{**dict(gradOutput=n, x=n, weight=None, bias=None, mean=fake(2, 2), rstd=fake(2, 2), groups=2), **kw})


def test_frequencies(monkeypatch):
    from arraymancer_amd import sequence_hip
    monkeypatch.setattr(sequence_hip, "toHip", lambda a: a)          # the values, without a device
    plain = sequence_hip.rotary_frequencies(8, base=100.0)
    assert np.allclose(plain, [1, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15)
    assert np.allclose(sequence_hip.rotary_frequencies(8, base=100.0, scaling="linear", factor=4), plain / 4, rtol=1e-15)
    grown = sequence_hip.rotary_frequencies(8, base=100.0, scaling="base", factor=4)
    assert grown[0] == 1 and np.isclose(grown[-1], plain[-1] / 4, rtol=1e-14)
    parts = sequence_hip.rotary_frequencies(64, scaling="parts", factor=8, context=2048)
    own = sequence_hip.rotary_frequencies(64)
    turns = 2048 * own / (2 * np.pi)
    assert np.array_equal(parts[turns > 32], own[turns > 32]) and np.allclose(parts[turns < 1], own[turns < 1] / 8, rtol=1e-15)
    assert (np.diff(parts) < 0).all()
    for kw in (dict(rot_dim=7), dict(rot_dim=0), dict(scaling="half"), dict(base=0.0), dict(factor=-1.0), dict(scaling="parts"), dict(rot_dim=2, scaling="base")):
        with pytest.raises(ValueError):
            sequence_hip.rotary_frequencies(**{**dict(rot_dim=8), **kw})


def _differences(f, x, grad, rng, tol):
    way = rng.normal(size=x.shape)
    way /= np.linalg.norm(way)
    h = 1e-5
    assert abs((f(x + h * way) - f(x - h * way)) / (2 * h) - (grad * way).sum()) <= tol


def test_the_definitions_gradients_against_differences():
    rng = np.random.default_rng(1)
    B, T, H, KH, dk, dv = 2, 6, 4, 2, 3, 5
    x = dict(q=rng.normal(size=(B, T, H, dk)), k=rng.normal(size=(B, T, KH, dk)), v=rng.normal(size=(B, T, KH, dv)), state=rng.normal(size=(B, H, dk, dv)))
    g, lengths = -1 / 2.0 ** np.arange(H), np.array([4, 6])
    go, gs = rng.normal(size=(B, T, H, dv)), rng.normal(size=(B, H, dk, dv))

    def loss(**kw):
        out, end = ref.attention(*[{**x, **kw}[n] for n in "qkv"], g, {**x, **kw}["state"], lengths, 0.7)
        return (out * go).sum() + (end * gs).sum()

    grads = ref.attention_backward(go, x["q"], x["k"], x["v"], g, x["state"], lengths, 0.7, gs)
    for name, grad in zip(("q", "k", "v", "state"), grads):
        _differences(lambda a: loss(**{name: a}), x[name], grad, rng, 1e-7)
    n = dict(x=rng.normal(size=(2, 3, 4, 6)) + 1, w=rng.normal(size=6), b=rng.normal(size=6))
    dy = rng.normal(size=n["x"].shape)
    for act in ("none", "relu", "silu"):
        for name, grad in zip(("x", "w", "b"), ref.norm_backward(dy, n["x"], n["w"], n["b"], 3, 1e-3, act)):
            _differences(lambda a: (ref.norm(*[{**n, name: a}[m] for m in "xwb"], 3, 1e-3, act) * dy).sum(), n[name], grad, rng, 1e-6)


def test_the_cpp_host_layer_builds():
    where = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
    res = subprocess.run(["make", "-C", where, "-B", "test_sequence"], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-3000:]
