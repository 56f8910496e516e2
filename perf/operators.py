"""Cases, plain forms and exact values of the sequence-mixing operators: rotary positions, linear attention with a decay for
each head (prompts, training, single tokens) and group normalisation with an activation over channels-last tensors.

`listed()` names the cases, `draw(rng)` gives more of the same ranges, `prepare` makes the inputs of one on the device, `run` is
one pass, `work` what that pass cannot do without and `exact` its result from the definition in 64 bits. With `own` false
`run` is written in elementary torch operations; with `own` true it makes the calls of arraymancer_amd on the same tensors.

Shapes: q [batch, tokens, heads, dk], k [batch, tokens, kv_heads, dk], v [batch, tokens, kv_heads, dv], state
[batch, heads, dk, dv]; query head h reads key / value head h // (heads / kv_heads). Images are [batch, height, width, channels].
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f64": torch.float64}


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of 32 requests, each at a place of its own in its text: latency
        dict(name="rotary_token", kind="rotary", backward=False, dtype="f32", batch=32, tokens=1, heads=16, dim=128, rotated=128,
             layout="half", context=32768, scale=1.0),
        # the queries of a batch of prompts: bandwidth
        dict(name="rotary_prompt", kind="rotary", backward=False, dtype="f32", batch=4, tokens=2048, heads=32, dim=128, rotated=128,
             layout="interleaved", context=2048, scale=1.0),
        # the gradient where only a part of the head turns, positions of a stretched context, odd length
        dict(name="rotary_backward_part", kind="rotary", backward=True, dtype="f64", batch=3, tokens=1023, heads=12, dim=80,
             rotated=48, layout="half", context=131072, scale=1.1),
        # one new token of two conversations: latency
        dict(name="step_two", kind="step", dtype="f32", batch=2, heads=16, kv_heads=16, dk=128, dv=128),
        # one new token of a full serving batch: the states' bandwidth
        dict(name="step_batch", kind="step", dtype="f32", batch=192, heads=16, kv_heads=16, dk=128, dv=128),
        # a batch of prompts, the largest
        dict(name="prompt_batch", kind="prompt", dtype="f32", batch=4, tokens=4096, heads=16, kv_heads=16, dk=128, dv=128, padded=False,
             state=False),
        # one long text that continues from a state: few heads, many tokens, odd length
        dict(name="prompt_long", kind="prompt", dtype="f32", batch=1, tokens=16391, heads=8, kv_heads=8, dk=64, dv=64, padded=False,
             state=True),
        # a padded batch with shared key / value heads and odd sizes, in 64 bits
        dict(name="prompt_padded", kind="prompt", dtype="f64", batch=5, tokens=777, heads=6, kv_heads=2, dk=48, dv=80, padded=True,
             state=True),
        # a training step through the layer: output and every gradient, key / value heads shared by four
        dict(name="train", kind="train", dtype="f32", batch=4, tokens=2048, heads=16, kv_heads=4, dk=64, dv=128, padded=False, state=False),
        # the norm of each head's output behind the attention, a batch of prompts
        dict(name="norm_heads", kind="norm", train=False, dtype="f32", batch=16384, height=1, width=1, channels=2048, groups=16,
             activation="silu", affine=True),
        # a convolution's output in training: forward pass and gradients
        dict(name="norm_images_train", kind="norm", train=True, dtype="f32", batch=16, height=64, width=64, channels=320, groups=32,
             activation="silu", affine=True),
        # the norm of each head for eight new tokens: latency
        dict(name="norm_token", kind="norm", train=False, dtype="f32", batch=8, height=1, width=1, channels=2048, groups=16,
             activation="none", affine=True),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotary", "step", "prompt", "train", "norm"])
    dtype = rng.choice(["f32", "f32", "f64"])
    if kind == "rotary":
        dim = 2 * rng.randint(16, 96)
        heads = rng.randint(1, 32)
        tokens = 1 if rng.random() < 0.25 else _spread(rng, 2, 4096)
        batch = max(1, min(_spread(rng, 1, 64), (1 << 24) // (tokens * heads * dim)))
        return dict(kind=kind, backward=rng.random() < 0.5, dtype=dtype, batch=batch, tokens=tokens, heads=heads, dim=dim,
                    rotated=dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2), layout=rng.choice(["half", "interleaved"]),
                    context=rng.choice([2048, 32768, 131072]), scale=rng.choice([1.0, 1.1]))
    if kind == "norm":
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        channels = groups * rng.randint(1, 1024 // groups)
        side = rng.choice([1, rng.randint(2, 64)])
        batch = max(1, min(_spread(rng, 1, 8192) if side == 1 else _spread(rng, 1, 32), (1 << 23) // (side * side * channels)))
        # no training through relu: next to 0 the rounding of z decides whether a gradient passes
        train = rng.random() < 0.5
        return dict(kind=kind, train=train, dtype=dtype, batch=batch, height=side, width=max(1, side - rng.randint(0, 1)),
                    channels=channels, groups=groups, activation=rng.choice(["none", "silu"] + ([] if train else ["relu"])),
                    affine=rng.random() < 0.8)
    kv_heads = rng.randint(1, 8)
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    dk, dv = rng.randint(16, 160), rng.randint(16, 160)
    if kind == "step":
        return dict(kind=kind, dtype=dtype, batch=_spread(rng, 1, 128), heads=heads, kv_heads=kv_heads, dk=dk, dv=dv)
    tokens = _spread(rng, 1, 8192 if kind == "prompt" else 2048)
    batch = max(1, min(_spread(rng, 1, 16), (1 << 22) // (tokens * heads * max(dk, dv))))
    return dict(kind=kind, dtype=dtype, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv,
                padded=rng.random() < 0.4, state=rng.random() < 0.5)


# ---------------------------------------------------------------------- inputs
def prepare(case, seed):
    dt = DTYPES[case["dtype"]]
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * scale + mean).to(dt)

    b = case["batch"]
    if case["kind"] == "rotary":
        t, n = case["tokens"], case["rotated"] // 2
        # frequencies 10000^(-i / n), the slow ones stretched by four as for a context longer than the trained one
        freq = torch.pow(10000.0, -torch.arange(n, device=DEVICE, dtype=torch.float64) / max(n, 1))
        if case["context"] > 2048:
            turns = 2048 * freq / (2 * math.pi)
            keep = ((turns - 1) / 31).clamp(0, 1)
            freq = freq * (keep + (1 - keep) / 4)
        first = torch.randint(0, max(1, case["context"] - t + 1), (b, 1), generator=gen, device=DEVICE)
        return dict(case=dict(case), x=normal(b, t, case["heads"], case["dim"]), freq=freq,
                    positions=(first + torch.arange(t, device=DEVICE)).contiguous())
    if case["kind"] == "norm":
        c = case["channels"]
        shape = (b, c) if case["height"] * case["width"] == 1 else (b, case["height"], case["width"], c)
        s = dict(case=dict(case), x=normal(*shape, scale=1.5, mean=0.25), weight=None, bias=None)
        if case["affine"]:
            s.update(weight=normal(c, scale=0.2, mean=1.0), bias=normal(c, scale=0.2))
        if case["train"]:
            s["grad"] = normal(*shape)
        return s
    h, kh, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    # a token's weight falls to 1/e within 4 tokens in the fastest head and 256 in the slowest
    reach = torch.exp2(torch.linspace(2, 8, h, device=DEVICE, dtype=torch.float64)) * torch.rand((h,), generator=gen, device=DEVICE).add(0.5)
    s = dict(case=dict(case), log_decay=(-1.0 / reach).to(dt), scale=dk ** -0.5)
    if case["kind"] == "step":
        s.update(q=normal(b, h, dk), k=normal(b, kh, dk), v=normal(b, kh, dv), state=normal(b, h, dk, dv))
        return s
    t = case["tokens"]
    s.update(q=normal(b, t, h, dk), k=normal(b, t, kh, dk), v=normal(b, t, kh, dv), state=None, lengths=None)
    if case["state"]:
        s["state"] = normal(b, h, dk, dv)
    if case["padded"]:
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=gen, device=DEVICE)
        s["lengths"][0] = t
    if case["kind"] == "train":
        s["grad"] = normal(b, t, h, dv)
        if case["state"]:
            s["grad_state"] = normal(b, h, dk, dv)
    return s


# ---------------------------------------------------------------------- plain forms
def _plain_rotary(s):
    c = s["case"]
    x, n = s["x"], c["rotated"] // 2
    angle = s["positions"].to(torch.float64)[:, :, None, None] * s["freq"]
    cos, sin = (torch.cos(angle) * c["scale"]).to(x.dtype), (torch.sin(angle) * c["scale"]).to(x.dtype)
    if c["backward"]:
        sin = -sin
    turned, rest = x[..., :2 * n], x[..., 2 * n:]
    if c["layout"] == "half":
        a, b = turned[..., :n], turned[..., n:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _plain_step(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    k, v = s["k"].repeat_interleave(group, 1), s["v"].repeat_interleave(group, 1)
    state = s["state"]
    state.mul_(torch.exp(s["log_decay"])[:, None, None]).add_(k[..., :, None] * v[..., None, :])
    return torch.matmul((s["q"] * s["scale"])[..., None, :], state)[..., 0, :], state


CHUNK = 64


def _plain_scan(q, k, v, decay, state, after):
    """o_i = sum over j <= i of e^(decay (i - j)) (q_i . k_j) v_j + e^(decay (i + after)) q_i state, and the state behind the last
    token, e^(decay tokens) state + sum_j e^(decay (tokens - after - j)) k_j v_j; arrays [batch, heads, tokens, .], in chunks:
    products within each chunk, one product over all chunks' sums for the states between them. after = 1 going forwards."""
    b, h, t, dk = q.shape
    dv = v.shape[-1]
    n = -(-t // CHUNK)
    pad = n * CHUNK - t
    if pad:
        # in front: a zero token there adds nothing to what follows
        q, k, v = (torch.nn.functional.pad(x, (0, 0, pad, 0)) for x in (q, k, v))
    q, k, v = (x.reshape(b, h, n, CHUNK, x.shape[-1]) for x in (q, k, v))
    at = torch.arange(CHUNK, device=q.device, dtype=q.dtype)
    d = decay[:, None, None]
    apart = at[:, None] - at[None, :]
    mask = torch.where(apart >= 0, torch.exp(d * apart.clamp(min=0)), 0)                      # [h, C, C]
    out = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * mask[:, None], v)
    own_part = torch.matmul((k * torch.exp(d * (CHUNK - after - at)[:, None])[:, None]).transpose(-1, -2), v)   # [b, h, n, dk, dv]
    ends = torch.arange(n + 1, device=q.device, dtype=q.dtype)
    between = ends[:, None] - 1 - ends[None, :n]
    carry = torch.where(between >= 0, torch.exp(d * CHUNK * between.clamp(min=0)), 0)         # [h, n + 1, n]
    states = torch.matmul(carry, own_part.reshape(b, h, n, dk * dv)).reshape(b, h, n + 1, dk, dv)
    if state is not None:
        # the padding in front lies between the given state and the first token: its share of the decay is left out
        states = states + torch.exp(decay[:, None] * (ends * CHUNK - pad).clamp(min=0))[:, :, None, None] * state[:, :, None]
    reach = torch.exp(d * (at + after)[:, None])[:, None]                                    # [h, 1, C, 1]
    inter = torch.matmul(q * reach, states[:, :, :n])
    if state is not None and pad:
        # first chunk: its token i is the (i - pad)-th behind the given state
        first = torch.exp(d * (at - pad + after).clamp(min=0)[:, None])
        inter = torch.cat([torch.matmul(q[:, :, :1] * first[:, None], states[:, :, :1]), inter[:, :, 1:]], 2)
    out = (out + inter).reshape(b, h, n * CHUNK, dv)[:, :, pad:]
    return out, states[:, :, n]


def _heads_first(x, group, live):
    x = x.permute(0, 2, 1, 3)
    if group > 1:
        x = x.repeat_interleave(group, 1)
    return x if live is None else torch.where(live, x, 0)


def _plain_attention(s):
    c = s["case"]
    t, group = c["tokens"], c["heads"] // c["kv_heads"]
    lengths, state, g = s["lengths"], s["state"], s["log_decay"]
    live, shift, back = None, None, None
    at = torch.arange(t, device=g.device)
    if lengths is not None:
        # every text is moved to the end of its row (zero tokens in front add nothing), and moved back afterwards
        shift = (at[None, :] - (t - lengths[:, None])) % t
        back = (at[None, :] + (t - lengths[:, None])) % t
        live = (at[None, :] < lengths[:, None])[:, None, :, None]

    def load(x, grouped):
        x = _heads_first(x, group if grouped else 1, live)
        return x if shift is None else torch.gather(x, 2, shift[:, None, :, None].expand_as(x))

    def store(x):
        return x if back is None else torch.where(live, torch.gather(x, 2, back[:, None, :, None].expand_as(x)), 0)

    def scan(q, k, v, st, after):
        """Behind a padded row's zero tokens the state has not decayed yet: it is given a decay that undoes theirs."""
        if st is None or lengths is None:
            return _plain_scan(q, k, v, g, st, after)
        out, end = _plain_scan(q, k, v, g, None, after)
        behind = (at[None, :] - (t - lengths[:, None]))[:, None, :]                         # place in the text, negative in front
        w = torch.where(behind >= 0, torch.exp(g[:, None] * (behind.clamp(min=0) + after).to(g.dtype)), 0)
        out = out + torch.matmul(q, st) * w[..., None]
        return out, end + st * torch.exp(g * lengths[:, None].to(g.dtype))[..., None, None]

    q, k, v = load(s["q"] * s["scale"], False), load(s["k"], True), load(s["v"], True)
    out, end = scan(q, k, v, state, 1)
    out = store(out).permute(0, 2, 1, 3)
    if c["kind"] == "prompt":
        return out, end
    do = load(s["grad"], False)
    turned = state.transpose(-1, -2) if state is not None else None
    dq, _ = scan(do, v, k, turned, 1)
    dq = dq * s["scale"]

    # from the last token to the first
    def reverse(x):
        return x.flip(2)

    ds = s.get("grad_state")
    if lengths is None:
        r = [reverse(x) for x in (q, k, v, do)]
        dv, dstate = _plain_scan(r[1], r[0], r[3], g, ds, 0)
        dk, _ = _plain_scan(r[2], r[3], r[0], g, ds.transpose(-1, -2) if ds is not None else None, 0)
    else:
        # reversed, a text begins its row and the zero tokens follow it; they are moved in front again
        turn = (at[None, :] + lengths[:, None]) % t
        undo = (at[None, :] - lengths[:, None]) % t

        def move(x, to):
            return torch.gather(x, 2, to[:, None, :, None].expand_as(x))

        r = [move(reverse(x), turn) for x in (q, k, v, do)]
        dv, dstate = scan(r[1], r[0], r[3], ds, 0)
        dk, _ = scan(r[2], r[3], r[0], ds.transpose(-1, -2) if ds is not None else None, 0)
        dv, dk = move(dv, undo), move(dk, undo)
    dv, dk = reverse(dv), reverse(dk)
    dq, dk, dv = (store(x) for x in (dq, dk, dv))
    if group > 1:
        dk, dv = (x.unflatten(1, (c["kv_heads"], group)).sum(2) for x in (dk, dv))
    got = [out, end] + [x.permute(0, 2, 1, 3) for x in (dq, dk, dv)]
    return got + [dstate] if state is not None else got


EPS = 1e-5


def _plain_norm(s):
    c = s["case"]
    x, g = s["x"], c["groups"]
    per = c["channels"] // g
    v = x.reshape(c["batch"], -1, g, per)
    mean = v.mean((1, 3), keepdim=True)
    rstd = ((v - mean).square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    xhat = (v - mean) * rstd
    z = xhat
    if c["affine"]:
        w, b = s["weight"].reshape(g, per), s["bias"].reshape(g, per)
        z = xhat * w + b
    sig = 1 / (1 + torch.exp(-z)) if c["activation"] == "silu" else None
    y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0), "silu": lambda: z * sig}[c["activation"]]().reshape(x.shape)
    if not c["train"]:
        return y
    dz = s["grad"].reshape(v.shape)
    if c["activation"] == "silu":
        dz = dz * (sig * (1 + z * (1 - sig)))
    dxhat = dz * w if c["affine"] else dz
    dx = rstd * (dxhat - dxhat.mean((1, 3), keepdim=True) - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
    dx = dx.reshape(x.shape)
    if not c["affine"]:
        return y, dx
    return y, dx, (dz * xhat).sum((0, 1)).reshape(-1), dz.sum((0, 1)).reshape(-1)


# ---------------------------------------------------------------------- the framework's calls
class _Lent:
    """A torch tensor's memory as the storage of a HipTensor."""
    __slots__ = ("ptr", "nelems", "itemsize", "owner")

    def __init__(self, t):
        self.ptr, self.nelems, self.itemsize, self.owner = t.data_ptr(), t.numel(), t.element_size(), t


class _View:
    """A HipTensor's memory as a torch tensor."""

    def __init__(self, t):
        self.owner = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": t.dtype.str, "data": (t.data_ptr(), False), "strides": None,
                                         "version": 2}


_NAMES = {torch.float32: "float32", torch.float64: "float64", torch.int64: "int64"}


def _hip(am, t):
    return None if t is None else am.HipTensor(am.Layout(tuple(t.shape), t.stride(), 0), _Lent(t), _NAMES[t.dtype])


def _torch(t):
    return None if t is None else torch.as_tensor(_View(t), device=DEVICE)


_library = []                     # the library's stream, once torch's work has joined it


def _join(am):
    """From the first call on torch works on the stream that the library puts all of its own work on, as in a program that uses both:
    what torch writes or reads of the tensors that the two lend to each other, and of memory that either takes again, is ordered with
    the library's calls by the stream itself. (Two streams with events between them cost every call 20 to 40 us.)"""
    am.sync()
    library = torch.cuda.ExternalStream(am.load_library().am_hip_stream())
    library.wait_stream(torch.cuda.current_stream())
    torch.cuda.set_stream(library)
    _library.append(library)


def _own(s):
    import arraymancer_amd as am

    if not _library:
        _join(am)
    c = s["case"]
    if c["kind"] == "rotary":
        call = am.rotary_backward if c["backward"] else am.rotary
        return _torch(call(_hip(am, s["x"]), _hip(am, s["positions"]), _hip(am, s["freq"]), layout=c["layout"], scale=c["scale"]))
    if c["kind"] == "norm":
        x, w, b = _hip(am, s["x"]), _hip(am, s["weight"]), _hip(am, s["bias"])
        if not c["train"]:
            return _torch(am.group_norm(x, w, b, c["groups"], eps=EPS, activation=c["activation"]))
        y, mean, rstd = am.group_norm_forward(x, w, b, c["groups"], eps=EPS, activation=c["activation"])
        grads = am.group_norm_backward(_hip(am, s["grad"]), x, w, b, mean, rstd, c["groups"], activation=c["activation"])
        return [_torch(t) for t in (y,) + grads if t is not None]
    q, k, v, g, state = (_hip(am, s[n]) for n in ("q", "k", "v", "log_decay", "state"))
    if c["kind"] == "step":
        return _torch(am.decay_attention_step(q, k, v, g, state, scale=s["scale"])), s["state"]
    lengths = _hip(am, s["lengths"])
    out, end = am.decay_attention(q, k, v, g, state=state, lengths=lengths, scale=s["scale"])
    if c["kind"] == "prompt":
        return _torch(out), _torch(end)
    grads = am.decay_attention_backward(_hip(am, s["grad"]), q, k, v, g, state=state, lengths=lengths, scale=s["scale"],
                                        gradState=_hip(am, s.get("grad_state")))
    return [_torch(t) for t in (out, end) + grads if t is not None]


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "norm": _plain_norm, "step": _plain_step, "prompt": _plain_attention,
            "train": _plain_attention}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------- least work
def work(case):
    size = {"f32": 4, "f64": 8}[case["dtype"]]
    b = case["batch"]
    if case["kind"] == "rotary":
        n = b * case["tokens"] * case["heads"]
        return dict(bytes=2 * n * case["dim"] * size + b * case["tokens"] * 8 + case["rotated"] * 4, flops=3 * n * case["rotated"])
    if case["kind"] == "norm":
        n = b * case["height"] * case["width"] * case["channels"]
        params = case["channels"] * (2 if case["affine"] else 0)
        # forward: x and y; training: x, y, the gradient and dx, the parameters and their gradients
        return dict(bytes=((4 if case["train"] else 2) * n + (2 if case["train"] else 1) * params) * size,
                    flops=(26 if case["train"] else 10) * n)
    h, kh, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    cell = b * h * dk * dv
    if case["kind"] == "step":
        return dict(bytes=(2 * cell + b * (h * (dk + dv) + kh * (dk + dv))) * size, flops=5 * cell)
    n = b * case["tokens"]
    rows = n * (h * (dk + dv) + kh * (dk + dv))      # q and the output, k and v
    given = cell if case["state"] else 0
    if case["kind"] == "prompt":
        return dict(bytes=(rows + given + cell) * size, flops=4 * n * h * dk * dv)
    # training: also the output's gradient, dq, dk and dv (and the states' gradients)
    return dict(bytes=(2 * rows + 3 * given + cell) * size, flops=14 * n * h * dk * dv)


# ---------------------------------------------------------------------- values in 64 bits, from the definitions
def _exact_rotary(s):
    c = s["case"]
    x, r = s["x"].double(), c["rotated"]
    angle = s["positions"].double()[..., None] * s["freq"]
    unit = torch.polar(torch.full_like(angle, c["scale"]), -angle if c["backward"] else angle)[:, :, None, :]
    out = x.clone()
    pairs = x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if c["layout"] == "half" else x[..., :r].unflatten(-1, (r // 2, 2))
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
    out[..., :r] = (turned.transpose(-1, -2) if c["layout"] == "half" else turned).flatten(-2)
    return out


def _exact_step(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    k, v = (s[n].double()[:, :, None].expand(-1, -1, group, -1).flatten(1, 2) for n in "kv")
    state = s["state"].double() * s["log_decay"].double().exp()[None, :, None, None] + torch.einsum("bhi,bhj->bhij", k, v)
    return torch.einsum("bhi,bhij->bhj", s["q"].double(), state) * s["scale"], state


def _exact_attention(s):
    """The recurrence itself, token by token: S <- e^g S + k v', o = scale q S; backwards R <- q do' + e^g R."""
    c = s["case"]
    b, t, h, kh = c["batch"], c["tokens"], c["heads"], c["kv_heads"]
    group, scale = h // kh, s["scale"]
    lam = s["log_decay"].double().exp()[None, :, None, None]
    live = torch.ones((b, t), device=DEVICE, dtype=torch.bool)
    if s["lengths"] is not None:
        live = torch.arange(t, device=DEVICE)[None] < s["lengths"][:, None]
    full = live.all(0).tolist()

    def row(name, i, grouped):
        x = s[name][:, i].double()
        return x[:, :, None].expand(-1, -1, group, -1).flatten(1, 2) if grouped else x

    def outer(x, y):
        return x[..., :, None] * y[..., None, :]

    def times(x, m):
        return (x[..., None, :] @ m)[..., 0, :]

    state = s["state"].double() if s["state"] is not None else torch.zeros((b, h, c["dk"], c["dv"]), device=DEVICE, dtype=torch.float64)
    train = c["kind"] == "train"
    out, dq = [], []
    for i in range(t):
        new = state * lam + outer(row("k", i, True), row("v", i, True))
        m = live[:, i, None, None]
        state = new if full[i] else torch.where(m[..., None], new, state)
        o = times(row("q", i, False), state) * scale
        out.append(o if full[i] else torch.where(m, o, 0))
        if train:
            d = times(row("grad", i, False), state.transpose(-1, -2)) * scale
            dq.append(d if full[i] else torch.where(m, d, 0))
    got = [torch.stack(out, 1), state]
    if not train:
        return got
    # what a token's state means for the outputs from it on; `carry` is its share of the token before
    carry = s["grad_state"].double() if s["state"] is not None else torch.zeros_like(state)
    dk, dv = [], []
    for i in reversed(range(t)):
        r = outer(row("q", i, False), row("grad", i, False)) * scale + carry
        m = live[:, i, None, None]
        a, d = times(row("v", i, True), r.transpose(-1, -2)), times(row("k", i, True), r)
        if not full[i]:
            a, d = torch.where(m, a, 0), torch.where(m, d, 0)
        dk.append(a.unflatten(1, (kh, group)).sum(2))
        dv.append(d.unflatten(1, (kh, group)).sum(2))
        carry = r * lam if full[i] else torch.where(m[..., None], r * lam, carry)
    got += [torch.stack(dq, 1), torch.stack(dk[::-1], 1), torch.stack(dv[::-1], 1)]
    return got + [carry] if s["state"] is not None else got


def _exact_norm(s):
    c = s["case"]
    n, ch, g = c["batch"], c["channels"], c["groups"]
    x = s["x"].double().reshape(n, -1, ch).transpose(1, 2).reshape(n, g, -1)             # a row for each group
    count = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / count
    var = (x - mean).pow(2).sum(-1, keepdim=True) / count
    root = torch.sqrt(var + EPS)
    xhat = ((x - mean) / root).reshape(n, ch, -1)
    w = s["weight"].double()[:, None] if c["affine"] else 1.0
    z = xhat * w + (s["bias"].double()[:, None] if c["affine"] else 0.0)
    y = z.clamp(min=0) if c["activation"] == "relu" else z / (1 + torch.exp(-z)) if c["activation"] == "silu" else z

    def back(a):
        return a.transpose(1, 2).reshape(s["x"].shape)

    if not c["train"]:
        return back(y)
    dz = s["grad"].double().reshape(n, -1, ch).transpose(1, 2)
    if c["activation"] == "silu":
        p = 1 / (1 + torch.exp(-z))
        dz = dz * (p + z * p * (1 - p))
    d = (dz * w).reshape(n, g, -1)
    h = xhat.reshape(n, g, -1)
    dx = (d * count - d.sum(-1, keepdim=True) - h * (d * h).sum(-1, keepdim=True)) / (count * root)
    got = [back(y), back(dx.reshape(n, ch, -1))]
    return got + [(dz * xhat).sum((0, 2)), dz.sum((0, 2))] if c["affine"] else got


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "norm": _exact_norm, "step": _exact_step, "prompt": _exact_attention,
            "train": _exact_attention}[case["kind"]](s)
