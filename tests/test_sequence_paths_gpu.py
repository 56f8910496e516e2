"""The sequence operators at the C interface's edges and along every way that their dispatch can take, on the device.

u = half a step of the element type. Attention is compared with its closed form (no recurrence) in float64; a result that is a
sum of products may be off by the roundings that a term passes, counted as in tests/test_sequence_gpu.py, times u times the sum
of the absolute terms."""
import numpy as np
import pytest

import sequence_closed as closed
import sequence_reference as ref
from arraymancer_amd._lib import last_error
from arraymancer_amd.sequence_hip import _rows
from conftest import DTYPES, seed_of
from test_sequence_gpu import attention_inputs, close, norm_bounds, norm_inputs, roundings, unit

pytestmark = pytest.mark.gpu


def strided(t, token_stride):
    """Pointer and strides of `t` [batch, tokens, heads, dim], with another token stride than its own."""
    p, b, _, h = _rows(t)
    return p, b, token_stride, h


@pytest.mark.parametrize("stride", [0, 1, 7, -3])
@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("dk,dv", [(8, 12), (64, 128), (7, 5)])
def test_a_single_tokens_stride_does_not_matter(hip, dk, dv, dt, stride):
    """With one token the token stride of an operand or a result leads nowhere, whatever it is: the bits of the packed call,
    forwards and backwards, and nothing beside the results."""
    B, H, KH = 3, 4, 4
    x = attention_inputs(hip, (B, 1, H, KH, dk, dv), dt, seed_of("one token", dk, dv, dt))
    d = {n: hip.toHip(a) for n, a in x.items() if n not in ("scale", "lengths")}
    want = hip.decay_attention(d["q"], d["k"], d["v"], d["g"], state=d["state"], scale=0.5)
    want += hip.decay_attention_backward(d["go"], d["q"], d["k"], d["v"], d["g"], state=d["state"], scale=0.5, gradState=d["gs"])
    got = [hip.toHip(np.full(t.shape, 7, DTYPES[dt])) for t in want]
    sizes = (B, 1, H, KH, dk, dv, 0.5, d["g"].data_ptr(), None)
    q, k, v, go = (strided(d[n], stride) for n in ("q", "k", "v", "go"))
    L = hip.load_library()
    s0 = _rows(d["state"])[:3]
    assert getattr(L, f"am_hip_decay_attention_{dt}")(*sizes, *q, *k, *v, *s0, *strided(got[0], stride), *_rows(got[1])[:3]) == 0, last_error()
    assert getattr(L, f"am_hip_decay_attention_backward_{dt}")(*sizes, *go, *q, *k, *v, *s0, *_rows(d["gs"])[:3], *(a for t in got[2:5] for a in strided(t, stride)),
                                                               *_rows(got[5])[:3]) == 0, last_error()
    for a, b in zip(got, want):
        assert np.array_equal(a.toCpu(), b.toCpu())


@pytest.mark.parametrize("dt", ["f32", "f64"])
def test_rotary_rounds_its_sines_once(hip, dt):
    """Pairs (0, 1) give back the sines and cosines themselves, those next to 0 among them: as good relatively as a double sine,
    then rounded to the result's type. The device's sine and cosine are good to 2 steps (4 u of a double), the product with the
    scale to 1 u, NumPy's to 1 step (2 u)."""
    T, n = 4096, 8
    rng = np.random.default_rng(31)
    pos = rng.integers(-10 ** 6, 10 ** 6, (1, T))
    freq = rng.uniform(0.01, 1.0, n)
    angle = pos.astype(np.float64)[..., None] * freq
    assert (np.abs(np.sin(angle)) < 1e-3).sum() > 5 and (np.abs(np.cos(angle)) < 1e-3).sum() > 5
    allowed = 7 * 2.0 ** -53 + (2.0 ** -24 if dt == "f32" else 0)
    x = np.concatenate([np.zeros((1, T, 1, n)), np.ones((1, T, 1, n))], -1).astype(DTYPES[dt])
    got = hip.rotary(hip.toHip(x), hip.toHip(pos), hip.toHip(freq)).toCpu()[:, :, 0].astype(np.float64)
    for a, b in ((got[..., :n], -np.sin(angle)), (got[..., n:], np.cos(angle))):
        off = np.abs(a - b) / np.abs(b)
        assert off.max() <= allowed, f"{off.max() / allowed:.2f} times what is allowed"


def slow_decays(tokens, count):
    """float32 log decays near -10^-6 whose e^{g tokens} lies nearly half a step from the next float: rounded once and used again
    and again it would pull to one side by about u / 2 every time."""
    g = (-1e-6 * (1 + np.arange(20000) / 20000)).astype(np.float32)
    e = np.exp(g.astype(np.float64) * tokens)
    off = np.abs(e.astype(np.float32).astype(np.float64) - e)
    return np.sort(g[off > 0.8 * 2.0 ** -25][:count])


def walk(n):
    """What n roundings of half a step at most, with no side, come to: six times their standard deviation, and 4 u for what follows."""
    return (6 * np.sqrt(n / 3) + 4) * 2.0 ** -24


def test_slow_decays_keep_a_prompts_state(hip):
    """A state that only decays, over 1024 chunks in one walk (512 heads fill the device: no segments)."""
    H, T, D = 512, 32768, 4
    g = slow_decays(32, H)
    assert len(g) == H
    rng = np.random.default_rng(41)
    s = (rng.uniform(0.5, 1, (1, H, D, D)) * rng.choice([-1, 1], (1, H, D, D))).astype(np.float32)
    nothing = hip.zeros((1, 1, 1, D), np.float32).broadcast((1, T, H, D))
    out, end = hip.decay_attention(nothing, nothing, nothing, hip.toHip(g), state=hip.toHip(s))
    del out
    want = s.astype(np.float64) * np.exp(g.astype(np.float64) * T)[None, :, None, None]
    close(end.toCpu(), want, walk(T // 32) * np.abs(want), "state")


# Which kernel takes a walk goes by its rows (up to 32, 64, 96, 128, 192, 256), its columns, the heads and tokens there are, and by
# whether rows are whole vectors of 16 bytes; a walk of dk rows and dv columns goes with one of dv rows and dk columns in the backward
# pass. Many heads, for workgroups of 128 columns (more than 64 columns, and work for every CU):
MANY = [(4, 130, 32, 16, dk, dv) for dk, dv in ((32, 96), (64, 128), (96, 128), (192, 256), (30, 66), (62, 90), (94, 126), (190, 254), (128, 72), (126, 70),
                                               (256, 192), (254, 190), (96, 32), (128, 64), (66, 30), (90, 62))]
# and few, for those of 64 columns (whose rows two wavefronts share from 128 on), all in segments
FEW = [(2, 197, 2, 1, dk, dv) for dk, dv in ((32, 64), (96, 40), (128, 64), (192, 60), (256, 24), (30, 62), (94, 34), (126, 62), (190, 54), (254, 22), (64, 32),
                                            (40, 96), (64, 192), (24, 256), (62, 30), (34, 94), (62, 126), (54, 190), (22, 254))]
# float64 has one form, of 64 columns
DOUBLE = [(2, 197, 2, 1, dk, dv) for dk, dv in ((32, 64), (96, 128), (192, 256), (31, 63), (95, 127), (191, 255), (64, 32), (128, 96), (256, 192), (63, 31),
                                               (127, 95), (255, 191))]


@pytest.mark.parametrize("size,dt", [(s, "f32") for s in MANY + FEW] + [(s, "f64") for s in DOUBLE], ids=str)
def test_every_kernel_of_decay_attention(hip, size, dt):
    """Prompt and gradients through every chunk kernel, from a state and with one, sequences of all lengths."""
    x = attention_inputs(hip, size, dt, seed_of("paths", size, dt))
    x["lengths"][0], x["lengths"][-1] = size[1], size[1] // 2
    d = {n: hip.toHip(a) for n, a in x.items() if n != "scale"}
    kw = dict(lengths=x["lengths"], scale=x["scale"])
    ab = {n: np.abs(a) for n, a in x.items() if n not in ("lengths", "scale", "g")}
    got = hip.decay_attention(d["q"], d["k"], d["v"], d["g"], state=d["state"], lengths=d["lengths"], scale=x["scale"])
    got += hip.decay_attention_backward(d["go"], d["q"], d["k"], d["v"], d["g"], state=d["state"], lengths=d["lengths"], scale=x["scale"], gradState=d["gs"])
    want, bound = (closed.attention(a["q"], a["k"], a["v"], x["g"], a["state"], **kw) +
                   closed.attention_backward(a["go"], a["q"], a["k"], a["v"], x["g"], a["state"], gs=a["gs"], **kw) for a in (x, ab))
    for name, a, b, m in zip(("out", "state", "dq", "dk", "dv", "dstate"), got, want, bound):
        close(a.toCpu(), b, roundings(size) * unit(DTYPES[dt]) * m, name)


# ---------------------------------------------------------------------- group norm's slabs
# Runs of memory too short for an image held in registers, or groups too large: whole rows of a slab, in vectors and singly.
SLABS = [((2, 3000, 4), 4), ((1, 4225, 24), 2), ((2, 2100, 7), 7)]


def chain(dt):
    """The roundings that a slab's sums pass. They run in double: of a lane's run of 64 rows, of up to 256 lanes, of up to 256 slabs
    a lane of the fold and of its 8 folds, 600 at most; in float only what follows them counts."""
    return 600 if dt == "f64" else 64


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups", SLABS, ids=str)
def test_slabs_without_parameters_and_of_a_large_mean(hip, shape, groups, dt):
    x, _, _, dy = norm_inputs(shape, dt, seed_of("slab mean", shape, dt), mean=300.0)
    by, bdx, _, _ = norm_bounds(x, None, None, dy, groups, 1e-3, dt, chain(dt))
    y, mean, rstd = hip.group_norm_forward(hip.toHip(x), None, None, groups, eps=1e-3)
    close(y.toCpu(), ref.norm(x, None, None, groups, 1e-3), by, "y")
    dx, dw, db = hip.group_norm_backward(hip.toHip(dy), hip.toHip(x), None, None, mean, rstd, groups)
    assert dw is None and db is None
    close(dx.toCpu(), ref.norm_backward(dy, x, None, None, groups, 1e-3)[0], bdx, "dx")


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups", SLABS, ids=str)
def test_slabs_far_out(hip, shape, groups, dt):
    """Weights that take silu far beyond the range of e^z on both sides; only one of the parameters' gradients wanted."""
    x, w, b, dy = norm_inputs(shape, dt, seed_of("slab far", shape, dt))
    w *= DTYPES[dt](300)
    bounds = norm_bounds(x, w, b, dy, groups, 1e-5, dt, chain(dt))
    X, W, B, DY = (hip.toHip(a) for a in (x, w, b, dy))
    y, mean, rstd = hip.group_norm_forward(X, W, B, groups, activation="silu")
    with np.errstate(over="ignore"):
        want = (ref.norm(x, w, b, groups, 1e-5, "silu"),) + ref.norm_backward(dy, x, w, b, groups, 1e-5, "silu")
    for name, a, r, bound in zip(("y", "dx", "dweight", "dbias"), (y,) + hip.group_norm_backward(DY, X, W, B, mean, rstd, groups, activation="silu"), want, bounds):
        close(a.toCpu(), r, bound, name)
    y, mean, rstd = hip.group_norm_forward(X, W, None, groups)
    dx, dw, db = hip.group_norm_backward(DY, X, W, None, mean, rstd, groups)
    bounds = norm_bounds(x, w, None, dy, groups, 1e-5, dt, chain(dt))
    want = ref.norm_backward(dy, x, w, None, groups, 1e-5)
    assert db is None
    close(y.toCpu(), ref.norm(x, w, None, groups, 1e-5), bounds[0], "y")
    close(dx.toCpu(), want[0], bounds[1], "dx")
    close(dw.toCpu(), want[1], bounds[2], "dweight")


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups", SLABS + [((3, 130, 48), 3), ((5, 7, 60), 4), ((4, 20, 512), 1)], ids=str)
def test_group_norm_of_rows_with_gaps(hip, shape, groups, dt):
    """Rows that lie apart, on 16-byte boundaries and off them, for x, for the gradient and for both, through slabs, images, teams and
    workgroups: nothing is copied first, and the result is that of packed operands up to the roundings of another order."""
    from arraymancer_amd.sequence_hip import _channels_last
    C = shape[-1]
    x, w, b, dy = norm_inputs(shape, dt, seed_of("gaps", shape, dt))
    W, B = hip.toHip(w), hip.toHip(b)

    def apart(a, front):
        wide = np.full(shape[:-1] + (C + 8,), 99, a.dtype)
        wide[..., front:front + C] = a
        t = hip.toHip(wide)[:, :, front:front + C]
        assert _channels_last(t)[0] is t and t.strides[1] == C + 8
        return t

    X, DY = hip.toHip(x), hip.toHip(dy)
    y, mean, rstd = hip.group_norm_forward(X, W, B, groups, activation="silu")
    want = [t.toCpu().astype(np.float64) for t in (y,) + hip.group_norm_backward(DY, X, W, B, mean, rstd, groups, activation="silu")]
    bounds = norm_bounds(x, w, b, dy, groups, 1e-5, dt, chain(dt))
    for front in (4, 1):
        for xs, ds in ((apart(x, front), DY), (X, apart(dy, front)), (apart(x, front), apart(dy, front))):
            y, m, r = hip.group_norm_forward(xs, W, B, groups, activation="silu")
            for a, c, t in zip((y,) + hip.group_norm_backward(ds, xs, W, B, m, r, groups, activation="silu"), want, bounds):
                close(a.toCpu(), c, 2 * t, f"front {front}")


@pytest.mark.parametrize("shape,groups", [((1, 40000, 2), 2), ((2, 4225, 24), 2), ((1, 70000, 3), 3)], ids=str)
def test_slabs_whose_first_elements_lie_far_from_the_rest(hip, shape, groups):
    """Elements around 1000 behind zeros, in the first row and at a few other places: in float64 the variance is as good as two passes
    make it. The sums pass up to 600 roundings (see `chain`); the subtraction of a run of 64 rows takes up to 64 times the three
    roundings of its operands: (600 + 3 * 64) u for the variance, half of it for rstd."""
    rng = np.random.default_rng(seed_of("pivot", shape))
    x = 1000 + rng.normal(size=shape)
    x[:, 0] = 0
    x[:, 64::9973] = 0
    x[:, 1::8192] = 2000
    _, mean, rstd = hip.group_norm_forward(hip.toHip(x), None, None, groups, eps=0.0)
    v = ref._grouped(x, groups).astype(np.longdouble)
    m = v.mean((1, 3), keepdims=True)
    want = 1 / np.sqrt(((v - m) ** 2).mean((1, 3)))
    u = 2.0 ** -53
    close(rstd.toCpu(), want.astype(np.float64), (600 + 3 * 64) / 2 * u * want.astype(np.float64), "rstd")
    close(mean.toCpu(), m[:, 0, :, 0].astype(np.float64), 600 * u * np.abs(v).mean((1, 3)).astype(np.float64), "mean")


# ---------------------------------------------------------------------- tensors larger than the caches keep
@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_past_the_caches(hip, dt, layout):
    """40 MB (80 in float64), read past the caches, give the bits of their parts, which are not."""
    B, T, H, D = 5, 997, 16, 128
    rng = np.random.default_rng(seed_of("far rotary", dt, layout))
    x, pos, freq = rng.normal(size=(B, T, H, D)).astype(DTYPES[dt]), rng.integers(0, 10 ** 5, (B, T)), hip.rotary_frequencies(96)
    whole = hip.rotary(hip.toHip(x), hip.toHip(pos), freq, layout=layout, scale=1.1).toCpu()
    for t in range(0, T, 250):
        part = hip.rotary(hip.toHip(np.ascontiguousarray(x[:, t:t + 250])), hip.toHip(np.ascontiguousarray(pos[:, t:t + 250])), freq, layout=layout, scale=1.1)
        assert np.array_equal(whole[:, t:t + 250], part.toCpu())


@pytest.mark.parametrize("dt", ["f32", "f64"])
def test_steps_past_the_caches(hip, dt):
    """States of 40 MB and more, one step of all against the steps of parts."""
    B, H, KH, D = 40, 16, 4, 128
    rng = np.random.default_rng(seed_of("far step", dt))
    mk = lambda *s: rng.normal(size=s).astype(DTYPES[dt])
    q, k, v, s, g = mk(B, H, D), mk(B, KH, D), mk(B, KH, D), mk(B, H, D, D), hip.toHip((-1 / 2.0 ** np.arange(H)).astype(DTYPES[dt]))
    state = hip.toHip(s)
    out = hip.decay_attention_step(hip.toHip(q), hip.toHip(k), hip.toHip(v), g, state, scale=0.1).toCpu()
    after = state.toCpu()
    for b in range(0, B, 10):
        part = hip.toHip(s[b:b + 10])
        # (fewer heads take narrower columns, and add up the rows in another order)
        got = hip.decay_attention_step(*(hip.toHip(a[b:b + 10]) for a in (q, k, v)), g, part, scale=0.1).toCpu()
        assert np.array_equal(after[b:b + 10], part.toCpu())
        bound = 0.1 * np.einsum("bhi,bhij->bhj", np.abs(q[b:b + 10]), np.abs(part.toCpu())).astype(np.float64)
        close(got, out[b:b + 10].astype(np.float64), 2 * (D + 2) * unit(DTYPES[dt]) * bound, "out")


@pytest.mark.parametrize("dt", ["f32", "f64"])
@pytest.mark.parametrize("shape,groups,parts", [((4200, 2048), 16, 4), ((2400, 3, 1280), 2, 4), ((6, 1000, 1000, 4), 4, 6)], ids=str)
def test_group_norm_past_the_caches(hip, shape, groups, parts, dt):
    """Teams, workgroups and slabs over more than 32 MB against the same samples in parts that fit; forwards without the statistics
    (which is what reads past the caches) and backwards. The parameters' gradients are added up from the parts'.
    Both sides' mean is off by chain u avg|x| (at most 1.04 deviations here) and rstd by chain u, xhat by their sum; dz moves with
    xhat by at most |dy w| / 2 times that, and is |dy| * 1.1 at most itself; a lane adds up 64 samples or 4 rows in the type."""
    shape = (shape[0] // (DTYPES[dt](0).itemsize // 4),) + shape[1:]
    parts = parts * 4 // DTYPES[dt](0).itemsize
    rng = np.random.default_rng(seed_of("far norm", shape, dt))
    C, T, u, n = shape[-1], DTYPES[dt], unit(DTYPES[dt]), chain(dt)
    x, dy = rng.standard_normal(shape, dtype=T) * T(2) + T(0.5), rng.standard_normal(shape, dtype=T)
    w, b = rng.standard_normal(C, dtype=T), rng.standard_normal(C, dtype=T)
    X, DY, W, B = (hip.toHip(a) for a in (x, dy, w, b))
    assert x.nbytes > 32 * 2 ** 20 >= x.nbytes // parts
    y = hip.group_norm(X, W, B, groups, activation="silu").toCpu()
    y2, mean, rstd = hip.group_norm_forward(X, W, B, groups, activation="silu")
    assert np.array_equal(y, y2.toCpu())
    dx, dw, db = (t.toCpu() for t in hip.group_norm_backward(DY, X, W, B, mean, rstd, groups, activation="silu"))
    sums, allowed = np.zeros((2, C)), np.zeros((2, C))
    for at in np.array_split(np.arange(shape[0]), parts):
        at = slice(at[0], at[-1] + 1)
        xp, dp = hip.toHip(x[at]), hip.toHip(dy[at])
        yp, m, r = hip.group_norm_forward(xp, W, B, groups, activation="silu")
        dxp, *grads = hip.group_norm_backward(dp, xp, W, B, m, r, groups, activation="silu")
        if at.stop == shape[0]:
            by, bdx, _, _ = norm_bounds(x[at], w, b, dy[at], groups, 1e-5, dt, n)
            close(yp.toCpu(), y[at].astype(np.float64), 2 * by, "y")
            close(dxp.toCpu(), dx[at].astype(np.float64), 2 * bdx, "dx")
        sums += [t.toCpu().astype(np.float64) for t in grads]
        xhat = (x[at].reshape(x[at].shape[0], -1, groups, C // groups) - m.toCpu()[:, None, :, None]) * r.toCpu()[:, None, :, None]
        h, d = np.abs(xhat).reshape(-1, C), np.abs(dy[at]).reshape(-1, C)
        off, wa = 2 * n * u * (h + T(1.04)), np.abs(w)
        allowed[0] += (d * (off * (1.1 + 0.5 * wa * h) + 128 * u * 1.1 * h)).sum(0, dtype=np.float64)
        allowed[1] += (d * (off * 0.5 * wa + 128 * u * 1.1)).sum(0, dtype=np.float64)
    close(dw, sums[0], allowed[0], "dweight")
    close(db, sums[1], allowed[1], "dbias")


# ---------------------------------------------------------------------- more than a launch holds
def test_group_norm_of_more_images_than_a_launch_holds(hip):
    """2^24 groups of 256 lanes each are 2^32 threads, which no launch may have: 2^18 samples of 64 groups, every one the same memory
    (the result has 34 GB). Forwards and backwards the first and the last are those of a single sample."""
    B, S, C, G = 2 ** 18, 128, 256, 64
    rng = np.random.default_rng(61)
    one = [hip.toHip(rng.standard_normal((1, S, C), dtype=np.float32)) for _ in range(2)]
    w = hip.toHip(rng.standard_normal(C, dtype=np.float32))
    x, dy = (t.broadcast((B, S, C)) for t in one)
    want = hip.group_norm_forward(one[0], w, w, G, activation="silu")
    y, mean, rstd = hip.group_norm_forward(x, w, w, G, activation="silu")
    for at in (slice(0, 1), slice(B - 1, B), slice(B // 2, B // 2 + 1)):
        assert np.array_equal(y[at].toCpu(), want[0].toCpu())
    assert (mean.toCpu() == want[1].toCpu()).all() and (rstd.toCpu() == want[2].toCpu()).all()
    del y
    grads = hip.group_norm_backward(one[1], one[0], w, w, *want[1:], G, activation="silu")
    dx, dw, db = hip.group_norm_backward(dy, x, w, w, mean, rstd, G, activation="silu")
    for at in (slice(0, 1), slice(B - 1, B), slice(B // 2, B // 2 + 1)):
        assert np.array_equal(dx[at].toCpu(), grads[0].toCpu())
    # 2^18 equal numbers are added in double: only the results are rounded, and the one sample's
    for a, b in ((dw, grads[1]), (db, grads[2])):
        assert (np.abs(a.toCpu() - B * b.toCpu().astype(np.float64)) <= 2 * 2.0 ** -24 * B * np.abs(b.toCpu())).all()


def test_shared_heads_are_added_up_over_several_launches(hip):
    """More gradients of keys than 2^16 workgroups take: with every head's own copy of keys and values, added up afterwards in the
    heads' order, the bits are the same."""
    B, T, H, dk, dv = 2, 140_000, 2, 65, 4
    assert B * T * dk > 2 ** 16 * 256
    rng = np.random.default_rng(62)
    mk = lambda *s: hip.toHip(rng.standard_normal(s, dtype=np.float32))
    q, k, v, go = mk(B, T, H, dk), mk(B, T, 1, dk), mk(B, T, 1, dv), mk(B, T, H, dv)
    g = hip.toHip(np.array([-0.5, -0.01], np.float32))
    _, dkey, dval, _ = hip.decay_attention_backward(go, q, k, v, g)
    _, keys, vals, _ = hip.decay_attention_backward(go, q, k.broadcast((B, T, H, dk)), v.broadcast((B, T, H, dv)), g)
    for a, b in ((dkey, keys), (dval, vals)):
        b = b.toCpu()
        assert np.array_equal(a.toCpu()[:, :, 0], b[:, :, 0] + b[:, :, 1])
