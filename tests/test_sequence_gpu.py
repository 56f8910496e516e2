"""Rotary positions, linear attention with decay and group norm on the device against their definitions in float64
(tests/sequence_reference.py).

Tolerances. u = half a step of the element type (eps / 2). A result that is a sum of products is off by at most
n * u * (the sum of the absolute values of its terms), where n counts the roundings a term passes: the definitions are run a
second time on absolute values to get those sums. The exponentials of the decays are good to 2 steps = 4 u and a product of
two of them and of its exponent adds 4 more."""
import os
import subprocess

import numpy as np
import pytest

import sequence_reference as ref
from arraymancer_amd.tensor_hip import _unary_into
from conftest import DTYPES, seed_of

pytestmark = pytest.mark.gpu


def unit(dtype):
    return np.finfo(dtype).eps / 2


def close(got, want, allowed, what=""):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == want.shape, (got.shape, want.shape)
    off = np.abs(got - want)
    assert np.isfinite(got).all(), f"{what}: values that are not finite"
    bad = off > allowed
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values off, worst {np.max(off / np.maximum(allowed, 1e-300)):.2f} times what is allowed"


# ---------------------------------------------------------------------- rotary
ROTARY_SIZES = [(1, 1, 1, 2, 2), (2, 3, 5, 80, 48), (1, 7, 3, 6, 4), (2, 5, 16, 128, 128), (3, 1, 4, 64, 64), (1, 33, 2, 10, 2),
                (2, 4, 9, 36, 0), (1, 300, 3, 64, 32)]


def freq_of(n):
    return 10000.0 ** (-np.arange(n, dtype=np.float64) / max(n, 1))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("size", ROTARY_SIZES, ids=str)
def test_rotary_and_its_gradient(hip, size, dt, layout):
    B, T, H, D, R = size
    rng = np.random.default_rng(seed_of("rotary", size, dt, layout))
    x = rng.normal(size=(B, T, H, D)).astype(DTYPES[dt])
    pos = rng.integers(-1000, 1_000_000, (B, T))
    freq, scale = freq_of(R // 2), 1.25
    dx, dp, df = hip.toHip(x), hip.toHip(pos), hip.toHip(freq)
    # the sines are good to 2 steps, times scale, times x, added: 8 u; in double the turns' rounding comes to it, 2^-54 of half a
    # turn: 12 u; for float results the angle is off by an ulp of 10^6
    a = ref.rotary(np.abs(x), np.zeros_like(pos), freq, layout, scale)
    partner = a.copy()
    f, s = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    partner[..., f], partner[..., s] = a[..., s], a[..., f]
    allowed = (a + partner) * (8 * unit(DTYPES[dt]) + 1e6 * 2.0 ** -52 if dt == "f32" else 12 * unit(DTYPES[dt]))
    for name, inverse in (("rotary", False), ("rotary_backward", True)):
        got = getattr(hip, name)(dx, dp, df, layout=layout, scale=scale).toCpu()
        close(got, ref.rotary(x, pos, freq, layout, scale, inverse), allowed, name)
        assert np.array_equal(got[..., R:], x[..., R:]), "the rest of the head is copied"
    # positions for all sequences at once, and none
    got = hip.rotary(dx, hip.toHip(pos[0].copy()), df, layout=layout, scale=scale).toCpu()
    close(got, ref.rotary(x, np.broadcast_to(pos[0], (B, T)), freq, layout, scale), allowed, "[tokens] positions")
    got = hip.rotary(dx, None, df, layout=layout, scale=scale).toCpu()
    close(got, ref.rotary(x, np.broadcast_to(np.arange(T), (B, T)), freq, layout, scale), allowed, "no positions")


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_of_views_and_in_place(hip, dt, layout):
    """Queries and keys side by side in one buffer, heads before tokens, one element off a 16-byte boundary, a reversed
    order of tokens, and the result over the operand: the bits are those of the contiguous call."""
    B, T, H, D, R = 2, 5, 4, 32, 32
    rng = np.random.default_rng(seed_of("rotary views", dt, layout))
    x = rng.normal(size=(B, T, H, D)).astype(DTYPES[dt])
    pos, freq = hip.toHip(rng.integers(0, 5000, (B, T))), hip.rotary_frequencies(R)
    want = hip.rotary(hip.toHip(x), pos, freq, layout=layout).toCpu()
    wide = hip.toHip(np.concatenate([x, x + 1], axis=2))
    assert np.array_equal(hip.rotary(wide[:, :, :H], pos, freq, layout=layout).toCpu(), want)
    swapped = hip.toHip(np.ascontiguousarray(x.transpose(0, 2, 1, 3))).permute(0, 2, 1, 3)
    assert np.array_equal(hip.rotary(swapped, pos, freq, layout=layout).toCpu(), want)
    odd = hip.toHip(np.concatenate([np.zeros((B, T, H, 1), x.dtype), x], axis=3))[:, :, :, 1:]
    assert np.array_equal(hip.rotary(odd, pos, freq, layout=layout).toCpu(), want)
    back = hip.toHip(np.ascontiguousarray(x[:, ::-1]))[:, ::-1]
    assert np.array_equal(hip.rotary(back, pos, freq, layout=layout).toCpu(), want)
    last = hip.toHip(np.ascontiguousarray(x.transpose(0, 1, 3, 2))).permute(0, 1, 3, 2)      # no unit stride: copied first
    assert np.array_equal(hip.rotary(last, pos, freq, layout=layout).toCpu(), want)
    inside = wide[:, :, :H]
    assert hip.rotary_into(inside, inside, pos, freq, layout=layout) is inside
    host = wide.toCpu()
    assert np.array_equal(host[:, :, :H], want) and np.array_equal(host[:, :, H:], x + 1), "in place, and nothing beside it"
    some = hip.rotary_frequencies(12)                          # a part of the head in place, and into another tensor's view
    part = hip.rotary(hip.toHip(x), pos, some, layout=layout).toCpu()
    here, other = hip.toHip(x), hip.toHip(np.concatenate([x, x], axis=3))
    hip.rotary_into(here, here, pos, some, layout=layout)
    hip.rotary_into(other[:, :, :, D:], hip.toHip(x), pos, some, layout=layout)
    assert np.array_equal(here.toCpu(), part)
    assert np.array_equal(other.toCpu()[..., D:], part) and np.array_equal(other.toCpu()[..., :D], x)


def test_rotary_keeps_far_positions(hip):
    """10^12 positions on, a float angle would be noise; the angle is the product in double, reduced without loss."""
    freq = freq_of(32)
    pos = np.array([[10 ** 12 + 7, -(10 ** 11) - 3, 2 ** 40]])
    x = np.random.default_rng(5).normal(size=(1, 3, 2, 64))
    angle = pos.astype(np.float64)[..., None] * freq
    c, s = np.cos(angle)[:, :, None], np.sin(angle)[:, :, None]
    want = np.concatenate([x[..., :32] * c - x[..., 32:] * s, x[..., 32:] * c + x[..., :32] * s], -1)
    got = hip.rotary(hip.toHip(x), hip.toHip(pos), hip.toHip(freq)).toCpu()
    # what is left of the turns is good to a few 2^-54 of half a turn (pi), both sines to a step or two, values up to 4, two terms
    assert np.abs(got - want).max() < 64 * 2.0 ** -53
    got32 = hip.rotary(hip.toHip(x.astype(np.float32)), hip.toHip(pos), hip.toHip(freq)).toCpu()
    # 10^12 * 2^-53 of an angle in double, then float's own roundings
    assert np.abs(got32 - want).max() < 4 * (10 ** 12 * 2.0 ** -52 + 8 * 2.0 ** -24) * np.abs(x).max()


# ---------------------------------------------------------------------- linear attention
#               batch tokens heads kv dk dv
ATTENTION = [(1, 1, 1, 1, 1, 1), (2, 5, 2, 1, 3, 7), (1, 63, 2, 2, 16, 16), (1, 64, 1, 1, 64, 64), (2, 65, 4, 2, 32, 48), (3, 33, 3, 1, 20, 130),
             (1, 200, 2, 2, 128, 128), (2, 31, 2, 1, 256, 40), (1, 97, 1, 1, 72, 256), (5, 2, 6, 3, 64, 96), (1, 32, 1, 1, 128, 17)]


def attention_inputs(hip, size, dt, seed):
    B, T, H, KH, dk, dv = size
    rng = np.random.default_rng(seed)
    mk = lambda *s: rng.normal(size=s).astype(DTYPES[dt])
    reach = 2.0 ** np.linspace(0, 7, H)
    return dict(q=mk(B, T, H, dk), k=mk(B, T, KH, dk), v=mk(B, T, KH, dv), g=(-1 / reach).astype(DTYPES[dt]), state=mk(B, H, dk, dv),
                go=mk(B, T, H, dv), gs=mk(B, H, dk, dv), lengths=rng.integers(0, T + 1, B), scale=dk ** -0.5)


def roundings(size):
    """What a term of an attention sum passes: a dot product of the operands, the sums over the tokens and the heads that
    share, the exponentials, the scale."""
    B, T, H, KH, dk, dv = size
    return max(dk, dv) + T + H // KH + 16


def check_attention(hip, size, dt, x, given, padded, grads):
    d = {n: hip.toHip(a) for n, a in x.items() if n != "scale"}
    state, gs = (x["state"], x["gs"]) if given else (None, None)
    dstate, dgs = (d["state"], d["gs"]) if given else (None, None)
    lengths, dlen = (x["lengths"], d["lengths"]) if padded else (None, None)
    kw = dict(lengths=lengths, scale=x["scale"])
    tol = roundings(size) * unit(DTYPES[dt])
    ab = {n: np.abs(a) for n, a in x.items() if n not in ("lengths", "scale", "g")}
    bound = ref.attention(ab["q"], ab["k"], ab["v"], x["g"], ab["state"] if given else None, **kw)
    out, end = hip.decay_attention(d["q"], d["k"], d["v"], d["g"], state=dstate, lengths=dlen, scale=x["scale"])
    want = ref.attention(x["q"], x["k"], x["v"], x["g"], state, **kw)
    close(out.toCpu(), want[0], tol * bound[0], "out")
    close(end.toCpu(), want[1], tol * bound[1], "state")
    if given:
        assert np.array_equal(d["state"].toCpu(), x["state"]), "the state that went in is as it was"
    if not grads:
        return
    got = hip.decay_attention_backward(d["go"], d["q"], d["k"], d["v"], d["g"], state=dstate, lengths=dlen, scale=x["scale"], gradState=dgs)
    want = ref.attention_backward(x["go"], x["q"], x["k"], x["v"], x["g"], state, gs=gs, **kw)
    bound = ref.attention_backward(ab["go"], ab["q"], ab["k"], ab["v"], x["g"], ab["state"] if given else None, gs=ab["gs"] if given else None, **kw)
    for name, a, b, m in zip(("dq", "dk", "dv", "dstate"), got, want, bound):
        if a is None:
            assert name == "dstate" and not given
            continue
        close(a.toCpu(), b, tol * m, name)


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("size", ATTENTION, ids=str)
def test_decay_attention_and_its_gradients(hip, size, dt):
    x = attention_inputs(hip, size, dt, seed_of("attention", size, dt))
    check_attention(hip, size, dt, x, given=True, padded=False, grads=True)
    check_attention(hip, size, dt, x, given=False, padded=False, grads=True)


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("size", [(5, 37, 2, 1, 24, 20), (4, 130, 3, 3, 64, 64), (3, 1, 2, 2, 8, 8)], ids=str)
def test_decay_attention_of_a_padded_batch(hip, size, dt):
    """Lengths 0, 1, the whole row, and beyond both ends; NaN and infinities behind the sequences reach nothing."""
    x = attention_inputs(hip, size, dt, seed_of("padded", size, dt))
    T = size[1]
    x["lengths"][:] = ([0, 1, T, T + 9, -4] + [T // 2] * size[0])[:size[0]]
    for b, n in enumerate(np.clip(x["lengths"], 0, T)):
        for name, bad in (("q", np.nan), ("k", np.inf), ("v", np.nan), ("go", -np.inf)):
            x[name][b, n:] = 0
    clean = {n: a.copy() if isinstance(a, np.ndarray) else a for n, a in x.items()}
    for b, n in enumerate(np.clip(x["lengths"], 0, T)):
        for name, bad in (("q", np.nan), ("k", np.inf), ("v", np.nan), ("go", -np.inf)):
            x[name][b, n:] = bad
    check_attention(hip, size, dt, clean, given=True, padded=True, grads=True)
    d, c = ({n: hip.toHip(a) for n, a in s.items() if n != "scale"} for s in (x, clean))
    run = lambda s: hip.decay_attention(s["q"], s["k"], s["v"], s["g"], state=s["state"], lengths=s["lengths"], scale=0.5)
    back = lambda s: hip.decay_attention_backward(s["go"], s["q"], s["k"], s["v"], s["g"], state=s["state"], lengths=s["lengths"], scale=0.5, gradState=s["gs"])
    for a, b in zip(run(d) + back(d), run(c) + back(c)):
        assert np.array_equal(a.toCpu(), b.toCpu())


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("size", [(2, 321, 4, 2, 64, 128), (2, 260, 8, 8, 64, 126), (1, 1411, 2, 1, 24, 40), (1, 9001, 1, 1, 8, 12)], ids=str)
def test_decay_attention_in_segments(hip, size, dt):
    """Long enough to be cut into segments: states between them in vectors, in single elements, over many slots; a sequence that
    ends within the first segments and one without tokens."""
    x = attention_inputs(hip, size, dt, seed_of("segments", size, dt))
    check_attention(hip, size, dt, x, given=True, padded=False, grads=True)
    for short in (0, 70):
        x["lengths"] = np.full(size[0], size[1], np.int64)
        x["lengths"][-1] = short
        check_attention(hip, size, dt, x, given=True, padded=True, grads=True)


@pytest.mark.parametrize("dt", ["f32", "f64"])
def test_decay_attention_of_no_tokens_and_of_extreme_decays(hip, dt):
    x = attention_inputs(hip, (2, 0, 2, 1, 6, 5), dt, 3)
    d = {n: hip.toHip(a) for n, a in x.items() if n not in ("scale", "lengths")}
    out, end = hip.decay_attention(d["q"], d["k"], d["v"], d["g"], state=d["state"])
    assert out.shape == (2, 0, 2, 5) and np.array_equal(end.toCpu(), x["state"])
    assert not hip.decay_attention(d["q"], d["k"], d["v"], d["g"])[1].toCpu().any()
    got = hip.decay_attention_backward(d["go"], d["q"], d["k"], d["v"], d["g"], state=d["state"], gradState=d["gs"])
    assert [t.shape for t in got[:3]] == [(2, 0, 2, 6), (2, 0, 1, 6), (2, 0, 1, 5)] and np.array_equal(got[3].toCpu(), x["gs"])
    # no decay at all, a decay that forgets everything, and one that underflows within a few tokens
    size = (1, 70, 3, 3, 16, 16)
    x = attention_inputs(hip, size, dt, 4)
    x["g"][:] = [0.0, -np.inf, -40.0]
    check_attention(hip, size, dt, x, given=True, padded=False, grads=True)


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("dk", [32, 30])
def test_decay_attention_of_reversed_views(hip, dt, dk):
    """Tokens stored last to first (negative strides), and one token's key standing for all (stride 0), forwards and backwards,
    with lengths: the bits of the contiguous call."""
    B, T, H, dv = 3, 75, 2, 34
    x = attention_inputs(hip, (B, T, H, H, dk, dv), dt, seed_of("reversed", dt, dk))
    x["lengths"][:] = [75, 41, 64]
    d = {n: hip.toHip(a) for n, a in x.items() if n != "scale"}
    back = lambda a: hip.toHip(np.ascontiguousarray(a[:, ::-1]))[:, ::-1]
    r = {n: back(x[n]) for n in ("q", "k", "v", "go")}

    def both(q, k, v, go):
        kw = dict(state=d["state"], lengths=d["lengths"], scale=0.3)
        return [t.toCpu() for t in hip.decay_attention(q, k, v, d["g"], **kw) + hip.decay_attention_backward(go, q, k, v, d["g"], gradState=d["gs"], **kw)]

    for a, b in zip(both(r["q"], r["k"], r["v"], r["go"]), both(d["q"], d["k"], d["v"], d["go"])):
        assert np.array_equal(a, b)
    one = d["k"][:, 0:1].broadcast((B, T, H, dk))
    same = hip.toHip(np.ascontiguousarray(np.broadcast_to(x["k"][:, :1], (B, T, H, dk))))
    for a, b in zip(both(d["q"], one, d["v"], d["go"]), both(d["q"], same, d["v"], d["go"])):
        assert np.array_equal(a, b)


def test_the_state_may_be_carried_in_place(hip):
    """state_out over state_in and grad_state_in over grad_state_out, which the C interface allows, in one segment and in many."""
    from arraymancer_amd.sequence_hip import _rows
    L = hip.load_library()
    for B, T, H, KH, dk, dv in ((2, 40, 2, 1, 16, 24), (1, 3000, 2, 2, 32, 32)):
        x = attention_inputs(hip, (B, T, H, KH, dk, dv), "f32", 12)
        d = {n: hip.toHip(a) for n, a in x.items() if n not in ("scale", "lengths")}
        out, end = hip.decay_attention(d["q"], d["k"], d["v"], d["g"], state=d["state"])
        grads = hip.decay_attention_backward(d["go"], d["q"], d["k"], d["v"], d["g"], state=d["state"], gradState=d["gs"])
        state, gs = hip.toHip(x["state"]), hip.toHip(x["gs"])
        mine = [hip.empty(t.shape, np.float32) for t in (out,) + grads[:3]]
        sizes = (B, T, H, KH, dk, dv, 1.0, d["g"].data_ptr(), None)
        q, k, v, go = (_rows(d[n]) for n in ("q", "k", "v", "go"))
        assert L.am_hip_decay_attention_f32(*sizes, *q, *k, *v, *_rows(state)[:3], *_rows(mine[0]), *_rows(state)[:3]) == 0
        assert L.am_hip_decay_attention_backward_f32(*sizes, *go, *q, *k, *v, *_rows(d["state"])[:3], *_rows(gs)[:3], *_rows(mine[1]), *_rows(mine[2]),
                                                     *_rows(mine[3]), *_rows(gs)[:3]) == 0
        for a, b in zip(mine + [state, gs], (out,) + grads[:3] + (end, grads[3])):
            assert np.array_equal(a.toCpu(), b.toCpu())


def far_view(hip, base, shape, strides, offset=0):
    from arraymancer_amd import Layout
    from arraymancer_amd.tensor_hip import HipTensor
    return HipTensor(Layout(shape, strides, offset), base.storage, base.dtype)


def test_operands_farther_apart_than_32_bits(hip):
    """Sequences 2^31 elements apart, and tokens 2^26 apart (32 of them do not fit a 32-bit offset): the bits of packed ones."""
    base = hip.empty((2 ** 31 + 2 ** 20,), np.float32)
    B, T, H, D = 2, 34, 1, 32
    rng = np.random.default_rng(21)
    host = {n: rng.normal(size=(B, T, H, D)).astype(np.float32) for n in ("q", "k", "v", "go")}
    near = {n: hip.toHip(a) for n, a in host.items()}
    g = hip.toHip(np.array([-0.05], np.float32))
    apart = {n: far_view(hip, base, (B, T, H, D), (2 ** 31, H * D, D, 1), i * T * H * D) for i, n in enumerate(host)}
    wide = {n: far_view(hip, base, (1, T - 2, H, D), (0, 2 ** 26, D, 1), 2 ** 15 + i * 64) for i, n in enumerate(host)}
    freq = hip.rotary_frequencies(D)
    for views, rows in ((apart, slice(0, T)), (wide, slice(0, T - 2))):
        n = views["q"].shape[0]
        packed = {m: hip.toHip(np.ascontiguousarray(a[:n, rows])) for m, a in host.items()}
        for m in views:
            _unary_into("copy", views[m], packed[m])
        got = hip.decay_attention(views["q"], views["k"], views["v"], g) + hip.decay_attention_backward(views["go"], views["q"], views["k"], views["v"], g)[:3] + \
            (hip.rotary(views["q"], None, freq), hip.decay_attention_step(*(views[m][:, 3].squeeze(1) for m in "qkv"), g, hip.zeros((n, H, D, D), np.float32)))
        want = hip.decay_attention(packed["q"], packed["k"], packed["v"], g) + hip.decay_attention_backward(packed["go"], packed["q"], packed["k"], packed["v"], g)[:3] + \
            (hip.rotary(packed["q"], None, freq), hip.decay_attention_step(*(packed[m][:, 3].squeeze(1) for m in "qkv"), g, hip.zeros((n, H, D, D), np.float32)))
        tol = 64 * unit(np.float32)
        for a, b in zip(got, want):     # (whole vectors and single elements take other kernels: rounding apart, not bits)
            a, b = a.toCpu(), b.toCpu()
            assert np.abs(a - b).max() <= tol * np.abs(b).max()
    rows = far_view(hip, base, (2, 40, 48), (2 ** 31, 48, 1), 11)
    x = rng.normal(size=(2, 40, 48)).astype(np.float32)
    _unary_into("copy", rows, hip.toHip(x))
    assert np.array_equal(hip.group_norm(rows, None, None, 4).toCpu(), hip.group_norm(far_view(hip, hip.toHip(np.concatenate([x.reshape(-1)[:11], x.reshape(-1)])), (2, 40, 48), (1920, 48, 1), 11), None, None, 4).toCpu())


@pytest.mark.parametrize("dt", ["f32", "f64"])
def test_decay_attention_of_views(hip, dt):
    """Queries, keys and values side by side in one buffer, heads before tokens, rows off a 16-byte boundary, one key head
    broadcast to all heads, states that are slices of a larger one."""
    B, T, H, dk, dv = 2, 45, 4, 32, 32
    size = (B, T, H, H, dk, dv)
    x = attention_inputs(hip, size, dt, seed_of("attention views", dt))
    d = {n: hip.toHip(a) for n, a in x.items() if n not in ("scale", "lengths")}
    want = [t.toCpu() for t in hip.decay_attention(d["q"], d["k"], d["v"], d["g"], state=d["state"])]
    fused = hip.toHip(np.concatenate([x["q"], x["k"], x["v"]], axis=2))
    q, k, v = (fused[:, :, i * H:(i + 1) * H] for i in range(3))
    pool = hip.toHip(np.stack([x["state"] * 0, x["state"]], axis=1))
    got = hip.decay_attention(q, k, v, d["g"], state=pool[:, 1].squeeze(1))
    for a, b in zip(got, want):
        assert np.array_equal(a.toCpu(), b)
    swap = lambda a: hip.toHip(np.ascontiguousarray(a.transpose(0, 2, 1, 3))).permute(0, 2, 1, 3)
    got = hip.decay_attention(swap(x["q"]), swap(x["k"]), swap(x["v"]), d["g"], state=d["state"])
    for a, b in zip(got, want):
        assert np.array_equal(a.toCpu(), b)
    shift = lambda a: hip.toHip(np.concatenate([a[..., :1], a], axis=-1))[:, :, :, 1:]
    got = hip.decay_attention(shift(x["q"]), shift(x["k"]), shift(x["v"]), d["g"], state=d["state"])
    for a, b in zip(got, want):
        assert np.array_equal(a.toCpu(), b)
    one = hip.decay_attention(d["q"], d["k"][:, :, 0:1].broadcast((B, T, H, dk)), d["v"], d["g"])[0].toCpu()
    same = hip.decay_attention(d["q"], hip.toHip(np.repeat(x["k"][:, :, :1], H, axis=2)), d["v"], d["g"])[0].toCpu()
    assert np.array_equal(one, same)


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("size", [(1, 9, 2, 2, 64, 64), (3, 6, 4, 2, 17, 33), (2, 40, 2, 1, 128, 96), (1, 3, 1, 1, 256, 256), (2, 4, 3, 3, 5, 1)], ids=str)
def test_steps_continue_a_prompt(hip, size, dt):
    """A prompt, then one token at a time from its state: each step against the definition, and the states agree."""
    B, T, H, KH, dk, dv = size
    x = attention_inputs(hip, size, dt, seed_of("steps", size, dt))
    head = T // 2
    want, last = ref.attention(x["q"], x["k"], x["v"], x["g"], x["state"], scale=x["scale"])
    ab = {n: np.abs(x[n]) for n in ("q", "k", "v", "state")}
    bound, last_bound = ref.attention(ab["q"], ab["k"], ab["v"], x["g"], ab["state"], scale=x["scale"])
    tol = roundings(size) * unit(DTYPES[dt])
    d = {n: hip.toHip(x[n]) for n in ("q", "k", "v", "g", "state")}
    out, state = hip.decay_attention(d["q"][:, :head], d["k"][:, :head], d["v"][:, :head], d["g"], state=d["state"], scale=x["scale"])
    if head:
        close(out.toCpu(), want[:, :head], tol * bound[:, :head], "prompt")
    for t in range(head, T):
        o = hip.decay_attention_step(*(d[n][:, t].squeeze(1) for n in "qkv"), d["g"], state, scale=x["scale"])
        close(o.toCpu(), want[:, t], tol * bound[:, t], f"token {t}")
    close(state.toCpu(), last, tol * last_bound, "state")


def test_a_step_leaves_the_rest_of_a_state_pool_alone(hip):
    rng = np.random.default_rng(9)
    pool = rng.normal(size=(5, 3, 2, 8, 12)).astype(np.float32)      # [slot, layer, heads, dk, dv]
    mk = lambda *s: rng.normal(size=s).astype(np.float32)
    q, k, v, g = mk(2, 2, 8), mk(2, 2, 8), mk(2, 2, 12), np.array([-0.1, -1.0], np.float32)
    d = hip.toHip(pool)
    part = d[1:5:2, 1].squeeze(1)
    out = hip.decay_attention_step(hip.toHip(q), hip.toHip(k), hip.toHip(v), hip.toHip(g), part)
    own = hip.toHip(np.ascontiguousarray(pool[1:5:2, 1]))
    same = hip.decay_attention_step(hip.toHip(q), hip.toHip(k), hip.toHip(v), hip.toHip(g), own)
    after = d.toCpu()
    assert np.array_equal(out.toCpu(), same.toCpu()) and np.array_equal(after[1:5:2, 1], own.toCpu())
    after[1:5:2, 1] = pool[1:5:2, 1]
    assert np.array_equal(after, pool)


# ---------------------------------------------------------------------- group norm
#           shape, groups
NORMS = [((1, 1), 1), ((3, 8), 2), ((5, 2048), 16), ((2, 7, 5, 30), 3), ((2, 16, 16, 40), 8), ((1, 64, 63, 10), 1), ((4, 3, 128), 32),
         ((700, 24), 4), ((1, 9000), 1), ((2, 3, 5000), 1), ((3, 40, 41, 320), 32), ((6, 1, 1, 64), 64), ((1, 300, 1030), 2), ((2, 70, 70, 3), 3)]


# many rows, whose group fits a workgroup's registers: vectors of four, two and one, 256 to 1024 lanes with few rows and with 48,
# lanes and dies left over; just too large; runs too short; the fewest rows; many samples, held and in slabs
IMAGES = [((2, 40, 40, 96), 6), ((3, 33, 31, 90), 6), ((1, 47, 44, 54), 2), ((9, 26, 25, 112), 4), ((1, 20, 20, 1024), 8), ((2, 59, 58, 13), 1),
          ((1, 64, 63, 12), 1), ((1, 65, 65, 24), 2), ((5, 16, 16, 32), 4), ((2, 45, 45, 28), 7), ((2, 128, 48), 3), ((2, 127, 48), 3), ((3, 20, 20, 9), 3),
          ((1201, 130, 16), 2), ((600, 2100, 2), 2)]


def norm_inputs(shape, dt, seed, mean=0.5):
    rng = np.random.default_rng(seed)
    mk = lambda *s: rng.normal(size=s).astype(DTYPES[dt])
    C = shape[-1]
    return (rng.normal(size=shape) * 2 + mean).astype(DTYPES[dt]), mk(C) + DTYPES[dt](1), mk(C), mk(*shape)


def norm_bounds(x, w, b, dy, groups, eps, dt, chain=64):
    """Allowed errors of y and dx. The sums of a group pass at most `chain` roundings (32 in a lane, 8 folds, the division
    and what follows); so mean is off by chain u avg|x|, rstd by chain u relatively, xhat by the sum of both."""
    u = unit(DTYPES[dt])
    mean, rstd = ref.norm_stats(x, groups, eps)
    v = ref._grouped(np.abs(x.astype(np.float64)), groups)
    xhat = np.abs(ref._grouped(x.astype(np.float64), groups) - mean) * rstd
    off = (rstd * (chain * u * v.mean((1, 3), keepdims=True) + 2 * u * v) + chain * u * xhat).reshape(x.shape)
    wa, ba = (np.ones(x.shape[-1]) if w is None else np.abs(w)), (0.0 if b is None else np.abs(b))
    y = 1.2 * (off * wa + 8 * u * (xhat.reshape(x.shape) * wa + ba))         # |act'| <= 1.1
    # dz moves with z by |dy act''| <= |dy| / 2 * (its error), and is rounded itself
    d = np.abs(dy) * wa * (1.1 * chain * u + 0.6 * wa * off + 8 * u * (xhat.reshape(x.shape) * wa + ba))
    mag = ref._grouped(np.abs(dy) * wa * 1.1, groups)
    dg, h, o = ref._grouped(d, groups), xhat, ref._grouped(off, groups)
    avg = lambda a: a.mean((1, 3), keepdims=True)
    dx = rstd * (dg + avg(dg) + h * avg(dg * h + mag * o) + o * avg(mag * h) + chain * u * (mag + avg(mag) + h * avg(mag * h)))
    flat = lambda a: a.reshape(-1, x.shape[-1]).sum(0)
    return y, dx.reshape(x.shape), flat((d / np.maximum(wa, 1e-30)) * h.reshape(x.shape) + np.abs(dy) * 1.1 * off) + 4 * u * flat(np.abs(dy) * h.reshape(x.shape)), \
        flat(d / np.maximum(wa, 1e-30)) + 4 * u * flat(np.abs(dy))


@pytest.mark.parametrize("activation", ["none", "relu", "silu"])
@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups", NORMS + IMAGES, ids=str)
def test_group_norm_and_its_gradients(hip, shape, groups, dt, activation):
    x, w, b, dy = norm_inputs(shape, dt, seed_of("norm", shape, groups, dt, activation))
    eps = 1e-5
    if activation == "relu":
        # next to 0 the rounding of z decides whether a gradient passes: none where it could go either way
        mean, rstd = ref.norm_stats(x, groups, eps)
        z = ((ref._grouped(x.astype(np.float64), groups) - mean) * rstd).reshape(x.shape) * w + b
        dy[np.abs(z) < 1e-4] = 0
    by, bdx, bdw, bdb = norm_bounds(x, w, b, dy, groups, eps, dt)
    dx_, dw_, db_, ddy = (hip.toHip(a) for a in (x, w, b, dy))
    y, mean, rstd = hip.group_norm_forward(dx_, dw_, db_, groups, eps=eps, activation=activation)
    close(y.toCpu(), ref.norm(x, w, b, groups, eps, activation), by, "y")
    assert np.array_equal(y.toCpu(), hip.group_norm(dx_, dw_, db_, groups, eps=eps, activation=activation).toCpu())
    got = hip.group_norm_backward(ddy, dx_, dw_, db_, mean, rstd, groups, activation=activation)
    want = ref.norm_backward(dy, x, w, b, groups, eps, activation)
    for name, a, r, bound in zip(("dx", "dweight", "dbias"), got, want, (bdx, bdw, bdb)):
        close(a.toCpu(), r, bound, name)
    again = hip.group_norm_backward(ddy, dx_, dw_, db_, mean, rstd, groups, activation=activation)
    for a, c in zip(got, again):
        assert np.array_equal(a.toCpu(), c.toCpu()), "the sums have a fixed order"


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups", [((4, 48), 6), ((2, 33, 40, 24), 3)], ids=str)
def test_group_norm_without_parameters_and_of_a_large_mean(hip, shape, groups, dt):
    x, w, b, dy = norm_inputs(shape, dt, seed_of("norm mean", shape, dt), mean=300.0)
    eps = 1e-3
    by, bdx, _, _ = norm_bounds(x, None, None, dy, groups, eps, dt)
    y, mean, rstd = hip.group_norm_forward(hip.toHip(x), None, None, groups, eps=eps)
    close(y.toCpu(), ref.norm(x, None, None, groups, eps), by, "y")
    dx, dw, db = hip.group_norm_backward(hip.toHip(dy), hip.toHip(x), None, None, mean, rstd, groups)
    assert dw is None and db is None
    close(dx.toCpu(), ref.norm_backward(dy, x, None, None, groups, eps)[0], bdx, "dx")


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups", [((6, 40), 4), ((2, 60, 50, 16), 2)], ids=str)
def test_group_norm_activations_far_out(hip, shape, groups, dt):
    """Weights that take silu far beyond the range of e^z on both sides: saturated, finite, and exact where it is 0 or z. The
    float sigmoid is good to 4 steps, z itself to what the norm's own bounds say."""
    x, w, b, dy = norm_inputs(shape, dt, seed_of("far out", shape, dt))
    w *= DTYPES[dt](300)
    by, bdx, bdw, bdb = norm_bounds(x, w, b, dy, groups, 1e-5, dt)
    y, mean, rstd = hip.group_norm_forward(hip.toHip(x), hip.toHip(w), hip.toHip(b), groups, activation="silu")
    with np.errstate(over="ignore"):
        want = ref.norm(x, w, b, groups, 1e-5, "silu")
        grads = ref.norm_backward(dy, x, w, b, groups, 1e-5, "silu")
    assert (np.abs(want) > 200).any() and (want == 0).any() or dt == "f64"
    close(y.toCpu(), want, by, "y")
    got = hip.group_norm_backward(hip.toHip(dy), hip.toHip(x), hip.toHip(w), hip.toHip(b), mean, rstd, groups, activation="silu")
    for name, a, r, bound in zip(("dx", "dweight", "dbias"), got, grads, (bdx, bdw, bdb)):
        close(a.toCpu(), r, bound, name)


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups", [((3, 6, 5, 24), 4), ((2, 50, 50, 16), 2), ((2, 30, 40, 36), 2)], ids=str)
def test_group_norm_of_views(hip, shape, groups, dt):
    """Images with the channels first (copied), a slice of the channels, rows with a gap, one element off a boundary."""
    x, w, b, dy = norm_inputs(shape, dt, seed_of("norm views", shape, dt))
    W, Bv, G = hip.toHip(w), hip.toHip(b), hip.toHip(dy)
    y, mean, rstd = hip.group_norm_forward(hip.toHip(x), W, Bv, groups, activation="silu")
    want = [y.toCpu()] + [t.toCpu() for t in hip.group_norm_backward(G, hip.toHip(x), W, Bv, mean, rstd, groups, activation="silu")]
    first = hip.toHip(np.ascontiguousarray(x.transpose(0, 3, 1, 2))).permute(0, 2, 3, 1)
    wide = hip.toHip(np.concatenate([x, x], axis=3))[:, :, :, :shape[-1]]
    rows = hip.toHip(np.concatenate([x, x], axis=2))[:, :, :shape[2]]
    odd = hip.toHip(np.concatenate([x[..., :1], x], axis=3))[:, :, :, 1:]
    for name, v in (("first", first), ("wide", wide), ("rows", rows), ("odd", odd)):
        y, m, r = hip.group_norm_forward(v, W, Bv, groups, activation="silu")
        got = [y] + list(hip.group_norm_backward(G, v, W, Bv, m, r, groups, activation="silu"))
        tol = norm_bounds(x, w, b, dy, groups, 1e-5, dt)
        for a, c, t in zip(got, want, tol):
            close(a.toCpu(), c.astype(np.float64), 2 * t, name)


def test_group_norm_of_more_samples_than_its_scratch_holds(hip):
    """2100 samples of 8192 channels in one group: their sums take more than 256 MB, so the slabs run in two launches and the second
    adds to the parameters' gradients of the first."""
    B, S, C = 2100, 2, 8192
    rng = np.random.default_rng(91)
    x, dy = rng.standard_normal((B, S, C), dtype=np.float32) * np.float32(2), rng.standard_normal((B, S, C), dtype=np.float32)
    X, DY, w, b = hip.toHip(x), hip.toHip(dy), hip.toHip(np.ones(C, np.float32)), hip.toHip(np.zeros(C, np.float32))
    y, mean, rstd = hip.group_norm_forward(X, w, b, 1)
    dx, dw, db = (t.toCpu() for t in hip.group_norm_backward(DY, X, w, b, mean, rstd, 1))
    sums, sizes = np.zeros((2, C)), np.zeros((2, C))
    for n in range(0, B, 300):
        d = dy[n:n + 300].astype(np.float64)
        xhat = ref.norm(x[n:n + 300], None, None, 1, 1e-5)
        for i, a in enumerate((d * xhat, d)):
            sums[i] += a.sum((0, 1))
        sizes[0] += (np.abs(d) * (np.abs(xhat) + 1)).sum((0, 1))
        sizes[1] += np.abs(d).sum((0, 1))
    # xhat: mean, rstd (2), difference, product; the product with dy, four rows in float, the result: 10 u of |dy| (|xhat| + 1)
    close(dw, sums[0], 10 * 2.0 ** -24 * sizes[0], "dweight")
    close(db, sums[1], 5 * 2.0 ** -24 * sizes[1], "dbias")
    part = slice(2040, 2056)                                                 # on both sides of the seam
    by, bdx, _, _ = norm_bounds(x[part], None, None, dy[part], 1, 1e-5, "f32")
    close(y.toCpu()[part], ref.norm(x[part], None, None, 1, 1e-5), by, "y")
    close(dx[part], ref.norm_backward(dy[part], x[part], None, None, 1, 1e-5)[0], bdx, "dx")


@pytest.mark.parametrize("shape,groups", [((0, 8), 2), ((3, 0, 8), 4), ((0, 4, 4, 6), 1)], ids=str)
def test_group_norm_of_nothing(hip, shape, groups):
    x = np.zeros(shape, np.float32)
    w = np.ones(shape[-1], np.float32)
    y, mean, rstd = hip.group_norm_forward(hip.toHip(x), hip.toHip(w), hip.toHip(w), groups)
    assert y.shape == shape and mean.shape == (shape[0], groups)
    dx, dw, db = hip.group_norm_backward(hip.toHip(x), hip.toHip(x), hip.toHip(w), hip.toHip(w), mean, rstd, groups)
    assert dx.shape == shape and not dw.toCpu().any() and not db.toCpu().any()


# ---------------------------------------------------------------------- together
def layer(hip, p, x, B, T, H, D, keep=False):
    """dense -> rotary -> decay attention -> group norm of each head -> dense, on x [B * T, features]."""
    heads = lambda t: t.reshape(B, T, H, D)
    q, k, v = (heads(hip.linear(x, p[n])) for n in ("wq", "wk", "wv"))
    qr, kr = hip.rotary(q, None, p["freq"]), hip.rotary(k, None, p["freq"])
    o, state = hip.decay_attention(qr, kr, v, p["g"], scale=D ** -0.5)
    flat = o.reshape(B * T, H * D)
    y, mean, rstd = hip.group_norm_forward(flat, p["w"], p["b"], H, activation="silu")
    out = hip.linear(y, p["wo"])
    return (out, state, (qr, kr, v, flat, y, mean, rstd)) if keep else (out, state)


def layer_backward(hip, p, x, kept, dout, B, T, H, D):
    qr, kr, v, flat, y, mean, rstd = kept
    dy, dwo = hip.linear_backward(y, p["wo"], dout, with_bias=False)
    do, dw, db = hip.group_norm_backward(dy, flat, p["w"], p["b"], mean, rstd, H, activation="silu")
    dq, dk, dv, _ = hip.decay_attention_backward(do.reshape(B, T, H, D), qr, kr, v, p["g"], scale=D ** -0.5)
    dq, dk = hip.rotary_backward(dq, None, p["freq"]), hip.rotary_backward(dk, None, p["freq"])
    grads, dx = {"wo": dwo, "w": dw, "b": db}, None
    for n, g in (("wq", dq), ("wk", dk), ("wv", dv)):
        gx, grads[n] = hip.linear_backward(x, p[n], g.reshape(B * T, H * D), with_bias=False)
        dx = gx if dx is None else dx + gx
    return dx, grads


def layer_parameters(hip, rng, F, H, D, dtype):
    mk = lambda *s: (rng.normal(size=s) / np.sqrt(s[-1])).astype(dtype)
    host = dict(wq=mk(H * D, F), wk=mk(H * D, F), wv=mk(H * D, F), wo=mk(F, H * D), w=mk(H * D) + 1, b=mk(H * D),
                g=-1 / 2.0 ** np.linspace(1, 5, H))
    p = {n: hip.toHip(a.astype(dtype)) for n, a in host.items()}
    p["freq"] = hip.rotary_frequencies(D)
    return host, p


def test_a_layers_gradients_against_differences(hip):
    """The whole layer in float64: directional derivatives by central differences. The third derivative of a layer this
    size is of the order of the loss itself, so with h = 1e-4 the difference is good to about 1e-8 + 1e-15 / h."""
    B, T, F, H, D = 2, 37, 24, 2, 16
    rng = np.random.default_rng(77)
    host, p = layer_parameters(hip, rng, F, H, D, np.float64)
    x = rng.normal(size=(B * T, F))
    weight = rng.normal(size=(B * T, F))
    out, _, kept = layer(hip, p, hip.toHip(x), B, T, H, D, keep=True)
    dx, grads = layer_backward(hip, p, hip.toHip(x), kept, hip.toHip(weight), B, T, H, D)
    loss = lambda pp, xx: float((layer(hip, pp, hip.toHip(xx), B, T, H, D)[0].toCpu() * weight).sum())
    h = 1e-4
    for name in ("x", "wq", "wk", "wv", "wo", "w", "b"):
        base = x if name == "x" else host[name]
        way = rng.normal(size=base.shape)
        way /= np.linalg.norm(way)
        at = []
        for s in (h, -h):
            if name == "x":
                at.append(loss(p, x + s * way))
            else:
                at.append(loss({**p, name: hip.toHip(base + s * way)}, x))
        got = float(((dx if name == "x" else grads[name]).toCpu() * way).sum())
        want = (at[0] - at[1]) / (2 * h)
        assert abs(got - want) <= 1e-6 * max(1.0, abs(want)), (name, got, want)


def test_a_layers_prompt_then_tokens(hip):
    """The layer over a prompt, then token by token with the carried state and its own positions, equals the layer over all
    tokens."""
    B, T, F, H, D, head = 2, 20, 16, 2, 32, 13
    rng = np.random.default_rng(78)
    _, p = layer_parameters(hip, rng, F, H, D, np.float64)
    x = rng.normal(size=(B, T, F))
    whole, last = layer(hip, p, hip.toHip(x.reshape(B * T, F)), B, T, H, D)
    whole = whole.toCpu().reshape(B, T, F)
    out, state = layer(hip, p, hip.toHip(np.ascontiguousarray(x[:, :head]).reshape(B * head, F)), B, head, H, D)
    assert np.allclose(out.toCpu().reshape(B, head, F), whole[:, :head], rtol=0, atol=1e-12)
    for t in range(head, T):
        xt = hip.toHip(np.ascontiguousarray(x[:, t]))
        pos = hip.toHip(np.full((B, 1), t))
        q, k, v = (hip.linear(xt, p[n]).reshape(B, 1, H, D) for n in ("wq", "wk", "wv"))
        hip.rotary_into(q, q, pos, p["freq"])
        hip.rotary_into(k, k, pos, p["freq"])
        o = hip.decay_attention_step(q.reshape(B, H, D), k.reshape(B, H, D), v.reshape(B, H, D), p["g"], state, scale=D ** -0.5)
        y = hip.group_norm(o.reshape(B, H * D), p["w"], p["b"], H, activation="silu")
        assert np.allclose(hip.linear(y, p["wo"]).toCpu(), whole[:, t], rtol=0, atol=1e-12), t
    assert np.allclose(state.toCpu(), last.toCpu(), rtol=0, atol=1e-12)


def test_group_norm_behind_a_convolution(hip):
    """conv2d gives [batch, channels, height, width]; its permuted view goes in, and the gradient comes back through it."""
    rng = np.random.default_rng(79)
    img, kern = rng.normal(size=(2, 3, 9, 8)), rng.normal(size=(12, 3, 3, 3))
    w, b = rng.normal(size=12), rng.normal(size=12)
    conv = hip.conv2d(hip.toHip(img), hip.toHip(kern), None, padding=(1, 1))
    last = conv.permute(0, 2, 3, 1)
    y, mean, rstd = hip.group_norm_forward(last, hip.toHip(w), hip.toHip(b), 4, activation="silu")
    host = conv.toCpu().transpose(0, 2, 3, 1)
    assert np.allclose(y.toCpu(), ref.norm(host, w, b, 4, 1e-5, "silu"), rtol=0, atol=1e-12)
    dy = rng.normal(size=y.shape)
    dx, dw, db = hip.group_norm_backward(hip.toHip(dy), last, hip.toHip(w), hip.toHip(b), mean, rstd, 4, activation="silu")
    want = ref.norm_backward(dy, host, w, b, 4, 1e-5, "silu")
    for a, r in zip((dx, dw, db), want):
        assert np.allclose(a.toCpu(), r, rtol=0, atol=1e-11)


# ---------------------------------------------------------------------- graphs
def test_a_layer_in_a_graph(hip):
    """Prompt, backward pass and step recorded into graphs, replayed with eager work between: every replay gives the eager
    bits. Two graphs with the same operators live side by side."""
    B, T, F, H, D = 2, 150, 32, 2, 32
    rng = np.random.default_rng(80)
    _, p = layer_parameters(hip, rng, F, H, D, np.float32)
    xs = [hip.toHip(rng.normal(size=(B * T, F)).astype(np.float32)) for _ in range(2)]
    dout = hip.toHip(rng.normal(size=(B * T, F)).astype(np.float32))

    def copy(dst, src):
        _unary_into("copy", dst, src)

    def train(x, into):
        out, state, kept = layer(hip, p, x, B, T, H, D, keep=True)
        dx, grads = layer_backward(hip, p, x, kept, dout, B, T, H, D)
        for dst, src in zip(into, (out, state, dx, grads["wq"], grads["w"])):
            copy(dst, src)

    made, eager = [], []
    for x in xs:
        out, state, kept = layer(hip, p, x, B, T, H, D, keep=True)
        dx, grads = layer_backward(hip, p, x, kept, dout, B, T, H, D)
        eager.append([t.toCpu() for t in (out, state, dx, grads["wq"], grads["w"])])
        into = [hip.empty(t.shape, np.float32) for t in (out, state, dx, grads["wq"], grads["w"])]
        made.append((hip.Graph.record(lambda x=x, into=into: train(x, into)), into))
    for turn in range(4):
        for (g, into), want in zip(made, eager):
            g.launch()
            hip.group_norm(xs[turn % 2], None, None, 4)                    # the program's own work between
            for t, w in zip(into, want):
                assert np.array_equal(t.toCpu(), w), f"replay {turn}"
    # steps: the state moves on at every replay
    mk = lambda *s: rng.normal(size=s).astype(np.float32)
    q, k, v, gd, s0 = mk(B, H, D), mk(B, H, D), mk(B, H, D), np.array([-0.5, -0.1], np.float32), mk(B, H, D, D)
    d = [hip.toHip(a) for a in (q, k, v, gd)]
    live, mirror, res = hip.toHip(s0), hip.toHip(s0), hip.empty((B, H, D), np.float32)
    spare = hip.toHip(s0)

    def one_step():
        copy(res, hip.decay_attention_step(*d, live))

    g = hip.Graph.record(one_step)
    copy(live, spare)
    for turn in range(3):
        g.launch()
        want = hip.decay_attention_step(*d, mirror).toCpu()
        assert np.array_equal(res.toCpu(), want) and np.array_equal(live.toCpu(), mirror.toCpu()), f"step {turn}"


@pytest.mark.parametrize("shape,groups", [((3, 20, 20, 48), 3), ((600, 130, 16), 2), ((2, 70, 71, 24), 8)], ids=str)
def test_group_norm_of_images_in_a_graph(hip, shape, groups):
    """Held groups, many samples' sums in runs, and slabs, with the memory they take for the call, recorded twice and replayed in
    turn: the eager bits every time."""
    made = []
    for i in range(2):
        x, w, b, dy = (hip.toHip(a) for a in norm_inputs(shape, "f32", seed_of("norm graph", shape, i)))

        def train(into=None, x=x, w=w, b=b, dy=dy):
            y, mean, rstd = hip.group_norm_forward(x, w, b, groups, activation="silu")
            got = (y,) + hip.group_norm_backward(dy, x, w, b, mean, rstd, groups, activation="silu")
            if into is None:
                return got
            for dst, src in zip(into, got):
                _unary_into("copy", dst, src)

        eager = train()
        into = [hip.empty(t.shape, np.float32) for t in eager]
        made.append((hip.Graph.record(lambda train=train, into=into: train(into)), into, [t.toCpu() for t in eager], train))
    for turn in range(3):
        for g, into, want, train in made:
            g.launch()
            train()                                                          # the program's own work between
            for t, w in zip(into, want):
                assert np.array_equal(t.toCpu(), w), f"replay {turn}"


@pytest.mark.parametrize("dt", ["f32", "f64"])
def test_decay_attention_in_segments_in_a_graph(hip, dt):
    """Few heads over many tokens, key / value heads shared, padded, a state carried on: segments, their states and the shared heads'
    shares all lie in memory taken for the call."""
    x = attention_inputs(hip, (2, 515, 4, 2, 64, 48), dt, seed_of("segments graph", dt))
    x["lengths"][:] = (515, 131)
    d = {n: hip.toHip(a) for n, a in x.items() if n != "scale"}

    def train():
        out = hip.decay_attention(d["q"], d["k"], d["v"], d["g"], state=d["state"], lengths=d["lengths"], scale=x["scale"])
        return out + hip.decay_attention_backward(d["go"], d["q"], d["k"], d["v"], d["g"], state=d["state"], lengths=d["lengths"], scale=x["scale"],
                                                  gradState=d["gs"])

    eager = train()
    want = [t.toCpu() for t in eager]
    into = [hip.empty(t.shape, DTYPES[dt]) for t in eager]

    def record():
        for dst, src in zip(into, train()):
            _unary_into("copy", dst, src)

    g = hip.Graph.record(record)
    for turn in range(3):
        g.launch()
        train()
        for t, w in zip(into, want):
            assert np.array_equal(t.toCpu(), w), f"replay {turn}"


# ---------------------------------------------------------------------- the C++ host layer
def test_the_cpp_host_layer(hip):
    program = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_sequence")
    if not os.path.exists(program):
        pytest.fail("tests/cpp/test_sequence is not built (python -c 'import __graft_entry__ as g; g.build()')")
    res = subprocess.run([program], capture_output=True, text=True, timeout=60)
    print(res.stdout)
    assert res.returncode == 0 and " 0 failed" in res.stdout, res.stdout[-3000:] + res.stderr[-1000:]
