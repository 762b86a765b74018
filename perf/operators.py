"""Cases for timing the sequence operators: layer norm, rotary positions over several axes, and linear
attention with a decay for each head (whole sequences, their gradients, and single steps).

They are the parts of a trajectory encoder that mixes the frames of each vehicle: the sizes are those of the
vehicle batches (32 packs of about 300 vehicles, 100 frames, 96 hidden units in 6 heads of 16), of the node
tables of the graph benchmarks (1M x 256), and generic long sequences.  ``own`` false runs plain torch forms.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-5
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _framework():
    """This repository's package, imported where its operators run."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sldm-gnn_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import sldm_sage
    return sldm_sage


# ------------------------------------------------------------------ cases --
def _ln(rows, width, dtype, train):
    return dict(op="norm", rows=rows, width=width, dtype=dtype, train=train)


def _rot(batch, frames, heads, kv_heads, dim, sections, dtype, train, grid, interleaved):
    return dict(op="rotary", batch=batch, frames=frames, heads=heads, kv_heads=kv_heads, dim=dim,
                sections=sections, dtype=dtype, train=train, grid=grid, interleaved=interleaved)


def _att(batch, frames, heads, kv_heads, dk, dv, dtype, train, ragged, state):
    return dict(op="attention", batch=batch, frames=frames, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv,
                dtype=dtype, train=train, ragged=ragged, state=state)


def _step(batch, heads, kv_heads, dk, dv, dtype):
    return dict(op="step", batch=batch, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, dtype=dtype)


def listed():
    return [
        # one training step's norm over the vehicles of a batch: short enough that launches count
        dict(_ln(9600, 96, "f32", True), name="norm train vehicles"),
        # the node table of the 1M-node benchmark, trained in bf16
        dict(_ln(1_000_000, 256, "bf16", True), name="norm train nodes"),
        # a wide hidden state whose width divides by nothing
        dict(_ln(20_011, 1031, "bf16", True), name="norm train odd width"),
        # the whole vehicle batch in training: time, x and y on three axes of each 16-wide head
        dict(_rot(9600, 100, 6, 6, 16, "2,3,3", "f32", True, False, False), name="rotary train vehicles"),
        # one new frame of one scene's vehicles, as live data comes in
        dict(_rot(300, 1, 6, 6, 16, "2,3,3", "bf16", False, False, False), name="rotary one frame"),
        # a long sequence of grid tokens (time, height, width), shared key heads, read from one projection
        dict(_rot(2, 16384, 16, 4, 128, "16,24,24", "bf16", False, True, True), name="rotary long grid"),
        # the vehicle batch in training: many short sequences with small heads
        dict(_att(9600, 100, 6, 6, 16, 16, "f32", True, False, False), name="attention train vehicles"),
        # prompts of uneven lengths that go on from a kept state
        dict(_att(8, 4096, 16, 16, 64, 64, "bf16", False, True, True), name="attention ragged prompts"),
        # few heads and a very long axis, trained
        dict(_att(1, 32768, 8, 8, 128, 128, "bf16", True, False, False), name="attention train long"),
        # shared key and value heads, unequal odd-ish head sizes, a length that divides by nothing
        dict(_att(5, 1237, 8, 2, 48, 80, "f32", True, True, True), name="attention train shared heads"),
        # one token for each of many sequences
        dict(_step(512, 16, 16, 64, 64, "bf16"), name="step many"),
        # one new frame of one scene's vehicles
        dict(_step(40, 6, 6, 16, 16, "f32"), name="step few"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "attention", "attention", "step"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "norm":
        width = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, max(2, min(2_000_000, 200_000_000 // width)))
        return _ln(rows, width, dtype, rng.random() < 0.7)
    if op == "rotary":
        dim = 2 * _log_int(rng, 4, 64)
        pairs = rng.randint(max(1, dim // 4), dim // 2)
        cuts = sorted(rng.randint(0, pairs) for _ in range(rng.randint(0, 3)))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        kv = rng.choice([1, 2, 4, 6])
        heads = kv * rng.choice([1, 1, 2, 4])
        tokens = _log_int(rng, 1, max(2, 150_000_000 // (dim * (heads + kv))))
        batch = _log_int(rng, 1, tokens)
        return _rot(batch, max(1, tokens // batch), heads, kv, dim, ",".join(map(str, sections)), dtype,
                    rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    kv = rng.choice([1, 2, 3, 4, 6, 8])
    heads = kv * rng.choice([1, 1, 1, 2, 4])
    dk, dv = (rng.choice([16, 24, 32, 40, 64, 80, 96, 128]) for _ in range(2))
    if rng.random() < 0.6:
        dv = dk
    if op == "step":
        batch = _log_int(rng, 1, max(2, 60_000_000 // (heads * dk * dv)))
        return _step(batch, heads, kv, dk, dv, dtype)
    tokens = _log_int(rng, 64, max(128, 32_000_000 // (heads * max(dk, dv))))
    frames = _log_int(rng, 1, min(tokens, 32768))
    return _att(max(1, tokens // frames), frames, heads, kv, dk, dv, dtype, rng.random() < 0.6,
                rng.random() < 0.5, rng.random() < 0.5)


# ------------------------------------------------------------------ inputs --
def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _frequencies(sections):
    """One frequency ladder for each axis, in 64 bits."""
    f = [10000.0 ** (-j / n) for n in sections for j in range(n)]
    return torch.tensor(f, dtype=torch.float64, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    s = {"case": case}
    if case["op"] == "norm":
        n, w = case["rows"], case["width"]
        s["x"] = (randn(n, w, dtype=torch.float32) * 1.5 + 0.3).to(dt)
        s["weight"] = 1 + 0.2 * randn(w, dtype=torch.float32)
        s["bias"] = 0.1 * randn(w, dtype=torch.float32)
        if case["train"]:
            s["dy"] = randn(n, w)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
        return s
    b, h, hk = case["batch"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        t, d = case["frames"], case["dim"]
        sections = _sections(case)
        s["sections"], s["inv_freq"] = sections, _frequencies(sections)
        if case["train"]:
            s["q"], s["k"] = randn(b, t, h, d).requires_grad_(True), randn(b, t, hk, d).requires_grad_(True)
            s["dq"], s["dk"] = randn(b, t, h, d), randn(b, t, hk, d)
        else:  # both are read from the projection that made them
            both = randn(b, t, h + hk, d)
            s["q"], s["k"] = both[:, :, :h], both[:, :, h:]
        axes = len(sections)
        if case["grid"]:
            s["positions"] = torch.randint(0, 1 << 16, (b, t, axes), generator=g, device=DEV)
        else:  # frames and metres
            s["positions"] = (torch.rand((b, t, axes), generator=g, device=DEV) - 0.5) * 1000
        return s
    dk, dv = case["dk"], case["dv"]
    s["log_decay"] = torch.log1p(-torch.exp2(-2 - 6 * torch.rand(h, generator=g, device=DEV)))
    s["scale"] = dk ** -0.5
    if case["op"] == "step":
        s["q"], s["k"], s["v"] = randn(b, h, dk), randn(b, hk, dk), randn(b, hk, dv)
        s["state"] = randn(b, h, dk, dv, dtype=torch.float32)
        return s
    t = case["frames"]
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, t + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    s["state"] = randn(b, h, dk, dv, dtype=torch.float32) if case["state"] else None
    if case["train"]:
        s["q"], s["k"], s["v"] = randn(b, t, h, dk), randn(b, t, hk, dk), randn(b, t, hk, dv)
        s["do"] = randn(b, t, h, dv)
        s["dstate"] = randn(b, h, dk, dv, dtype=torch.float32)
        for name in ("q", "k", "v", "state"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    else:  # views of the projection that made them
        qkv = randn(b, t, h * dk + hk * (dk + dv))
        q, k, v = qkv.split([h * dk, hk * dk, hk * dv], -1)
        s["q"], s["k"], s["v"] = q.unflatten(-1, (h, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hk, dv))
    return s


# ------------------------------------------------------------- plain forms --
def _plain_norm(s):
    x, w, b = s["x"].float(), s["weight"], s["bias"]
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    xhat = c * rstd
    out = {"y": (xhat * w + b).to(s["x"].dtype)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        out |= {"dx": dx.to(s["x"].dtype), "dweight": (dy * xhat).sum(0), "dbias": dy.sum(0)}
    return out


def _rotate(x, cos, sin, pairs, interleaved):
    """Pairs (j, j + pairs), or (2j, 2j + 1), of the first 2 * pairs values turned by their angles."""
    f = x.float()
    turned, rest = f[..., :2 * pairs], f[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _plain_rotary(s):
    sections, mixed = s["sections"], s["case"]["interleaved"]
    axis = torch.repeat_interleave(torch.arange(len(sections), device=DEV), torch.tensor(sections, device=DEV),
                                   output_size=sum(sections))
    angle = (s["positions"].double()[..., axis] * s["inv_freq"])[..., None, :]
    cos, sin, n = angle.cos().float(), angle.sin().float(), sum(sections)
    out = {"q": _rotate(s["q"], cos, sin, n, mixed), "k": _rotate(s["k"], cos, sin, n, mixed)}
    if s["case"]["train"]:
        out |= {"dq": _rotate(s["dq"], cos, -sin, n, mixed), "dk": _rotate(s["dk"], cos, -sin, n, mixed)}
    return out


CHUNK = 64


def _chunks(x, n, heads):
    """[B, T, h, D] in 32 bits as [B, heads, n, CHUNK, D], zeros behind the end, shared heads repeated."""
    b, t, h, d = x.shape
    x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, n * CHUNK - t)).transpose(1, 2)
    x = x[:, :, None].expand(b, h, heads // h, n * CHUNK, d)
    return x.reshape(b, heads, n, CHUNK, d)


def _plain_attention(s):
    """The chunked form: products inside a chunk, and states between chunks, all chunks at once."""
    c, scale = s["case"], s["scale"]
    b, t, h, hk = c["batch"], c["frames"], c["heads"], c["kv_heads"]
    dk, dv = c["dk"], c["dv"]
    n = t // CHUNK + 1
    ld = s["log_decay"].view(h, 1, 1)
    lens = s["lengths"].long() if s["lengths"] is not None else torch.full((b,), t, device=DEV)
    kept = torch.arange(t, device=DEV) < lens[:, None]

    def masked(x):
        return torch.where(kept[:, :, None, None], x.detach(), 0)

    q, k, v = (_chunks(masked(s[m]), n, h) for m in ("q", "k", "v"))
    i = torch.arange(CHUNK, device=DEV)
    ahead = i[:, None] - i
    tri = torch.where(ahead >= 0, torch.exp(ld * ahead.clamp(min=0)), 0)[:, None]       # [h, 1, C, C]
    since = torch.exp(ld * (i[:, None] + 1))[:, None]                                   # g^(i + 1)
    until = torch.exp(ld * (CHUNK - 1 - i)[:, None])[:, None]                           # g^(C - 1 - j)
    p = (q @ k.transpose(-1, -2)) * tri * scale
    m = torch.arange(n, device=DEV)
    apart = m[:, None] - 1 - m
    between = torch.where(apart >= 0, torch.exp(ld * (CHUNK * apart.clamp(min=0))), 0)  # [h, n, n]
    kv = (k * until).transpose(-1, -2) @ v
    before = (between @ kv.reshape(b, h, n, dk * dv)).reshape(b, h, n, dk, dv)
    state = s["state"].detach() if s["state"] is not None else None
    if state is not None:
        before = before + torch.exp(ld * (CHUNK * m)[:, None])[..., None] * state[:, :, None]
    o = p @ v + scale * since * (q @ before)

    def whole(x, d, like):
        return x.reshape(b, h, n * CHUNK, d)[:, :, :t].transpose(1, 2).to(like.dtype)

    # the state behind each sequence's last token
    at, left = lens // CHUNK, lens % CHUNK
    rows = torch.arange(b, device=DEV)
    gap = (left[:, None] - 1 - i)[:, None]
    w = torch.where(gap >= 0, torch.exp(s["log_decay"].view(1, h, 1) * gap.clamp(min=0)), 0)[..., None]
    end = torch.exp(s["log_decay"] * left[:, None])[..., None, None] * before[rows, :, at]
    end = end + (k[rows, :, at] * w).transpose(-1, -2) @ v[rows, :, at]
    out = {"o": whole(o, dv, s["v"]), "state": end}
    if not c["train"]:
        return out

    do = _chunks(masked(s["do"]), n, h)
    dend = s["dstate"]
    dp = (do @ v.transpose(-1, -2)) * tri * scale
    dq = dp @ k + scale * since * (do @ before.transpose(-1, -2))
    qd = scale * (q * since).transpose(-1, -2) @ do
    after = (between.transpose(-1, -2) @ qd.reshape(b, h, n, dk * dv)).reshape(b, h, n, dk, dv)
    # the final state's gradient reaches token j of a sequence with g^(length - 1 - j)
    gap = (lens[:, None] - 1 - torch.arange(n * CHUNK, device=DEV)).view(b, 1, n, CHUNK, 1)
    w = torch.where(gap >= 0, torch.exp(s["log_decay"].view(1, h, 1, 1, 1) * gap.clamp(min=0)), 0)
    late = dend[:, :, None]
    dk_ = dp.transpose(-1, -2) @ q + until * (v @ after.transpose(-1, -2)) + w * (v @ late.transpose(-1, -2))
    dv_ = p.transpose(-1, -2) @ do + until * (k @ after) + w * (k @ late)

    def shared(x, d, like):
        x = x.reshape(b, hk, h // hk, n * CHUNK, d).sum(2)[:, :, :t]
        return x.transpose(1, 2).to(like.dtype)

    out |= {"dq": whole(dq, dk, s["q"]), "dk": shared(dk_, dk, s["k"]), "dv": shared(dv_, dv, s["v"])}
    if state is not None:
        first = torch.exp(ld * (CHUNK * m))[..., None]                                  # [h, 1, n, 1]
        out["dstate"] = (qd * first.transpose(1, 2).reshape(h, n, 1, 1)).sum(2) \
            + torch.exp(s["log_decay"] * lens[:, None])[..., None, None] * dend
    return out


def _plain_step(s):
    group = s["case"]["heads"] // s["case"]["kv_heads"]
    k, v = (s[m].float().repeat_interleave(group, 1) for m in ("k", "v"))
    state = s["state"].mul_(torch.exp(s["log_decay"])[:, None, None]).add_(k[..., :, None] * v[..., None, :])
    o = s["scale"] * (s["q"].float()[..., None, :] @ state)[..., 0, :]
    return {"o": o.to(s["v"].dtype), "state": state}


# ---------------------------------------------------------- the framework's --
def _own_norm(s):
    sage = _framework()
    y = sage.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _own_rotary(s):
    sage = _framework()
    q, k = sage.rotary_axes(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"],
                            interleaved=s["case"]["interleaved"])
    if not s["case"]["train"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_attention(s):
    sage = _framework()
    o, end = sage.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"], state=s["state"],
                                  lengths=s["lengths"])
    out = {"o": o, "state": end}
    if not s["case"]["train"]:
        return out
    leaves = [m for m in ("q", "k", "v", "state") if s[m] is not None]
    grads = torch.autograd.grad((o, end), [s[m] for m in leaves], (s["do"], s["dstate"]))
    return out | {"d" + m: g for m, g in zip(leaves, grads)}


def _own_step(s):
    sage = _framework()
    o = sage.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale=s["scale"])
    return {"o": o, "state": s["state"]}  # moved on in place, as by the plain form


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "attention": _own_attention, "step": _own_step}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "rotary": _plain_rotary, "attention": _plain_attention, "step": _plain_step}[op](state)


# -------------------------------------------------------------------- work --
def work(case):
    """Each input read once, each output written once; the products of the recurrence."""
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "norm":
        n, w = case["rows"], case["width"]
        if case["train"]:  # x, dy in; y, dx out
            return {"bytes": 4 * n * w * e + 16 * w, "flops": 18 * n * w}
        return {"bytes": 2 * n * w * e + 8 * w, "flops": 8 * n * w}
    b, h, hk = case["batch"], case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        t, d, sections = case["frames"], case["dim"], _sections(case)
        ways = 2 if case["train"] else 1
        return {"bytes": ways * 2 * b * t * (h + hk) * d * e + b * t * len(sections) * (8 if case["grid"] else 4),
                "flops": ways * 6 * b * t * (h + hk) * sum(sections)}
    dk, dv = case["dk"], case["dv"]
    if case["op"] == "step":
        return {"bytes": b * (h * (dk + dv) + hk * (dk + dv)) * e + 8 * b * h * dk * dv, "flops": 5 * b * h * dk * dv}
    t = case["frames"]
    tokens = b * t / (2 if case["ragged"] else 1)
    rows = tokens * (h * (dk + dv) + hk * (dk + dv)) * e
    states = 4 * b * h * dk * dv * (2 if case["state"] else 1)
    if not case["train"]:
        return {"bytes": rows + states, "flops": 4 * tokens * h * dk * dv}
    # the gradients read q, k, v and do and write dq, dk and dv
    back = tokens * (h * (2 * dk + dv) + hk * 2 * (dk + dv)) * e
    return {"bytes": rows + back + 2 * states, "flops": 14 * tokens * h * dk * dv}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x, w, b = (s[m].detach().double().requires_grad_(case["train"]) for m in ("x", "weight", "bias"))
        centred = x - x.sum(-1, keepdim=True) / case["width"]
        y = centred / torch.sqrt(centred.square().sum(-1, keepdim=True) / case["width"] + EPS) * w + b
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if op == "rotary":
        return _exact_rotary(s)
    h, group = case["heads"], case["heads"] // case["kv_heads"]
    decay = torch.exp(s["log_decay"].double())[:, None, None]
    up = {m: s[m].detach().double().repeat_interleave(1 if m in ("q", "do") else group, -2)
          for m in ("q", "k", "v", "do") if m in s}
    if op == "step":
        state = decay * s["state"].double() + up["k"][..., None] * up["v"][..., None, :]
        return {"o": s["scale"] * (up["q"][..., None] * state).sum(-2), "state": state}
    return _exact_attention(s, up, decay, h, group)


def _exact_rotary(s):
    """Complex numbers turned by exp(i * position * frequency)."""
    sections = s["sections"]
    pos = torch.cat([s["positions"][..., a:a + 1].double().expand(*s["positions"].shape[:-1], n)
                     for a, n in enumerate(sections)], -1)
    turn = torch.polar(torch.ones_like(pos), pos * s["inv_freq"])[..., None, :]
    n = sum(sections)

    def apply(x, turn):
        x = x.detach().double()
        at = torch.arange(2 * n, device=DEV).view((n, 2) if s["case"]["interleaved"] else (2, n))
        re, im = at.unbind(-1 if s["case"]["interleaved"] else 0)
        z = torch.complex(x[..., re], x[..., im]) * turn
        x[..., re], x[..., im] = z.real, z.imag
        return x

    out = {"q": apply(s["q"].clone(), turn), "k": apply(s["k"].clone(), turn)}
    if s["case"]["train"]:
        out |= {"dq": apply(s["dq"].clone(), turn.conj()), "dk": apply(s["dk"].clone(), turn.conj())}
    return out


def _exact_attention(s, up, decay, h, group):
    """The recurrence, one token after the other."""
    c = s["case"]
    b, t, dk, dv = c["batch"], c["frames"], c["dk"], c["dv"]
    lens = s["lengths"].long() if s["lengths"] is not None else torch.full((b,), t, device=DEV)
    alive = (torch.arange(t, device=DEV)[:, None] < lens).double()[..., None, None, None]    # [t, b, 1, 1, 1]
    up = {m: (x * alive[..., 0].transpose(0, 1)).transpose(0, 1).contiguous() for m, x in up.items()}
    factor = 1 + alive * (decay - 1)
    start = s["state"].detach().double() if s["state"] is not None else torch.zeros(b, h, dk, dv, device=DEV, dtype=torch.float64)
    state, train = start.clone(), c["train"]
    o = torch.zeros(t, b, h, dv, device=DEV, dtype=torch.float64)
    dq = torch.zeros(t, b, h, dk, device=DEV, dtype=torch.float64) if train else None
    for n in range(t):
        state.mul_(factor[n]).addcmul_(up["k"][n][..., None], up["v"][n][..., None, :])
        torch.matmul(up["q"][n][..., None, :], state, out=o[n][..., None, :])
        if train:
            torch.matmul(state, up["do"][n][..., None], out=dq[n][..., None])
    o.mul_(s["scale"])
    out = {"o": o.transpose(0, 1), "state": state}
    if not train:
        return out
    grad = s["dstate"].double()
    dk_, dv_ = torch.zeros_like(up["k"]), torch.zeros_like(up["v"])
    for n in range(t - 1, -1, -1):
        grad = grad.addcmul(up["q"][n][..., None], up["do"][n][..., None, :], value=s["scale"])
        torch.matmul(grad, up["v"][n][..., None], out=dk_[n][..., None])
        torch.matmul(up["k"][n][..., None, :], grad, out=dv_[n][..., None, :])
        grad = grad * factor[n]
    out |= {"dq": dq.mul_(s["scale"]).transpose(0, 1),
            "dk": dk_.view(t, b, h // group, group, dk).sum(3).transpose(0, 1),
            "dv": dv_.view(t, b, h // group, group, dv).sum(3).transpose(0, 1)}
    if s["state"] is not None:
        out["dstate"] = grad
    return out
