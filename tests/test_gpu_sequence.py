"""The sequence operators (layer norm, rotary positions over several axes, decay attention and its
single step; csrc/norm.hip, rotary.hip, decay.hip) against their definitions in 64 bits
(oracle/sequence_ref.py).

Tolerances.  Every bound is elementwise.  A value rounded to the output's type is off by u |y| with
u = eps / 2 of that type (bf16 2^-8, fp32 2^-24).  A sum of n products in fp32 is off by at most
(n + 1) 2^-24 times the sum of the products' magnitudes, which the oracle gives for the magnitudes of
the inputs ("mag").  Decay attention in bf16 rounds each entry of Q K^T o D once to bf16 (2^-8 mag) and
reads the state as two bf16 terms (2^-16 mag); its decay weights are products of powers 2^x of an fp32
x (each within (2 + |x|) 2^-24): T + 256 terms of 2^-24 cover the sums and the weights.
"""
from __future__ import annotations

import math

import pytest
import torch

from oracle import sequence_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def _within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by " \
        f"{float((off - bound)[bad].max()):.3g} at {bad.nonzero()[0].tolist()}"


# --------------------------------------------------------------- layer norm --
def _norm_bounds(x, w, b, dy, eps):
    """Elementwise bounds for y, dx, dweight, dbias of rows x (float64)."""
    u, n = U[x.dtype], x.size(-1)
    e32 = 2.0 ** -24
    xd, dyd = x.double(), dy.double()
    mean = xd.mean(-1, keepdim=True)
    rstd = ((xd - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = (xd - mean) * rstd
    # mean is off by (n + 1) e32 mean|x|; centred values and rstd inherit that
    dmean = (n + 2) * e32 * xd.abs().mean(-1, keepdim=True)
    rel = (n + 8) * e32 + 2 * dmean * rstd
    exhat = rstd * dmean + xhat.abs() * rel + 4 * e32 * xhat.abs()
    wa = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double().abs()
    ba = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double().abs()
    y = (xhat.abs() * wa + ba) * (u + 4 * e32) + exhat * wa
    g = dyd.abs() * wa
    gm, gxm = g.mean(-1, keepdim=True), (g * xhat.abs()).mean(-1, keepdim=True)
    parts = g + gm + xhat.abs() * gxm
    dx = rstd * (parts * (u + rel + (n + 12) * e32) + exhat * gxm + xhat.abs() * (g * exhat).mean(-1, keepdim=True))
    rows = x.numel() // n
    lead = tuple(range(x.dim() - 1))
    dw = (dyd.abs() * (exhat + xhat.abs() * (rows + 4) * e32)).sum(lead)
    db = (dyd.abs() * (rows + 4) * e32).sum(lead)
    return y, dx, dw, db


NORM_SHAPES = [(1, 1), (3, 5), (7, 8), (5, 17), (64, 96), (33, 100), (2, 3, 4, 16), (257, 256), (9, 1031), (130, 520),
               (6, 2049), (3, 4098), (5, 8192), (4, 8193), (0, 64), (2, 20000), (5000, 24),
               (70, 264), (300, 257), (41, 5000), (3, 6144), (600, 320), (23, 1536)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
def test_layer_norm(shape, dtype):
    from sldm_sage import layer_norm
    g = _gen(1)
    x = (_randn(g, *shape) * 2 + 0.5).to(dtype).requires_grad_(True)
    w = (1 + 0.3 * _randn(g, shape[-1])).requires_grad_(True)
    b = (0.2 * _randn(g, shape[-1])).requires_grad_(True)
    dy = _randn(g, *shape, dtype=dtype)
    y = layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    assert y.dtype == dtype and got[0].dtype == dtype and got[1].dtype == torch.float32
    want, grads = ref.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    bounds = _norm_bounds(x.detach(), w.detach(), b.detach(), dy, 1e-5)
    _within(y, want, bounds[0], "y")
    for name, a, e, t in zip(("dx", "dweight", "dbias"), got, grads, bounds[1:]):
        _within(a, e, t, name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_strides_and_parts(dtype):
    """Rows inside a larger tensor, transposed dims, an expanded gradient, single gradients, no affine."""
    from sldm_sage import layer_norm
    g = _gen(2)
    big = _randn(g, 40, 3, 70, dtype=dtype)
    for x in (big[:, 1, 3:36], big.transpose(0, 1)[..., 5:25], big.permute(2, 0, 1), big[:, :, 1::3]):
        w = _randn(g, x.size(-1)).requires_grad_(True)
        leaf = x.detach().requires_grad_(True)
        y = layer_norm(leaf, w)
        dy = _randn(g, x.size(-1), dtype=dtype).expand(x.shape)
        bounds = _norm_bounds(x, w.detach(), None, dy, 1e-5)
        want, (dx, dw, _) = ref.layer_norm(x, w.detach(), None, 1e-5, dy)
        _within(y, want, bounds[0], "y")
        gx, gw = torch.autograd.grad(y, (leaf, w), dy, retain_graph=True)
        _within(gx, dx, bounds[1], "dx")
        _within(gw, dw, bounds[2], "dweight")
        assert torch.equal(torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], gx)
        assert torch.equal(torch.autograd.grad(y, w, dy)[0], gw)
        _within(layer_norm(x, eps=0.1), ref.layer_norm(x, eps=0.1), _norm_bounds(x, None, None, dy, 0.1)[0], "plain")


def test_layer_norm_module_and_bf16_parameters():
    from sldm_sage import LayerNorm
    g = _gen(3)
    ref_mod = torch.nn.LayerNorm(48)
    mod = LayerNorm(48)
    mod.load_state_dict(ref_mod.state_dict(), strict=True)
    mod = mod.to(DEV).bfloat16()
    x = _randn(g, 11, 48, dtype=torch.bfloat16).requires_grad_(True)
    y = mod(x)
    y.sum().backward()
    assert mod.weight.grad.dtype == torch.bfloat16 and x.grad.dtype == torch.bfloat16
    want = ref.layer_norm(x.detach(), mod.weight.detach(), mod.bias.detach())
    _within(y, want, _norm_bounds(x.detach(), mod.weight.detach(), mod.bias.detach(), x.detach(), 1e-5)[0], "y")


def test_layer_norm_constant_and_far_rows():
    """Rows without variance (xhat 0) and rows far from zero; NaN and Inf stay in their rows."""
    from sldm_sage import layer_norm
    x = torch.randn(6, 96, generator=_gen(4)).to(DEV)
    x[0] = 3.0
    x[1] += 1e4
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    y = layer_norm(x)
    assert torch.equal(y[0], torch.zeros_like(y[0]))
    want = ref.layer_norm(x[[1, 4, 5]])
    _within(y[[1, 4, 5]], want, _norm_bounds(x[[1, 4, 5]], None, None, x[[1, 4, 5]], 1e-5)[0], "y")
    assert y[2].isnan().all() and y[3].isnan().all()


# ------------------------------------------------------------------- rotary --
ROTARY = [  # lead, Hq, Hk, D, sections, interleaved
    ((1, 1), 1, 1, 2, (1,), False), ((1, 1), 1, 1, 2, (1,), True), ((3, 5), 2, 1, 16, (2, 3, 3), False),
    ((2, 7), 6, 6, 16, (2, 3, 3), True), ((37,), 4, 2, 22, (1, 0, 8), False), ((2, 3, 5), 3, 3, 128, (16, 24, 24), True),
    ((4, 50), 16, 4, 64, (32,), False), ((2, 129), 2, 2, 40, (7, 6), False), ((2, 33), 1, 3, 30, (1, 1, 1, 1, 1, 1, 1, 1), True),
    ((1, 70), 2, 2, 1024, (512,), False), ((3, 0), 2, 2, 16, (8,), False), ((5, 9), 2, 1, 9, (3,), False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotary_axes(case, dtype):
    from sldm_sage import rotary_axes, rotary_frequencies
    lead, hq, hk, D, sections, mix = case
    g = _gen(5)
    q, k = _randn(g, *lead, hq, D, dtype=dtype).requires_grad_(True), _randn(g, *lead, hk, D, dtype=dtype).requires_grad_(True)
    pos = ((torch.rand((*lead, len(sections)), generator=g) - 0.5) * 1000).to(DEV)
    f = rotary_frequencies(sections, device=DEV)
    oq, ok = rotary_axes(q, k, pos, f, sections, interleaved=mix)
    gq, gk = _randn(g, *lead, hq, D, dtype=dtype), _randn(g, *lead, hk, D, dtype=dtype)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk))
    u = U[dtype]
    for what, got, x, inverse in (("q", oq, q, False), ("k", ok, k, False), ("dq", dq, gq, True), ("dk", dk, gk, True)):
        x = x.detach()
        want = ref.rotary(x, pos, f, sections, mix, inverse)
        # sine and cosine within 4 ulp of an angle rounded to fp32 (pi 2^-24), two products, a sum, the output
        P = sum(sections)
        both = torch.zeros_like(want)
        pair = (x[..., 0:2 * P:2].double().abs() + x[..., 1:2 * P:2].double().abs()) if mix else \
            (x[..., :P].double().abs() + x[..., P:2 * P].double().abs())
        if mix:
            both[..., 0:2 * P:2] = both[..., 1:2 * P:2] = pair
        else:
            both[..., :P] = both[..., P:2 * P] = pair
        _within(got, want, u * want.abs() + 12 * 2.0 ** -24 * both, what)
        assert torch.equal(got[..., 2 * P:], x[..., 2 * P:])       # columns no axis turns


@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_rotary_position_types_and_far_positions(ptype):
    """Far positions: an angle of 2e6 (16e6 for whole numbers) keeps its place on the circle."""
    from sldm_sage import rotary_axes, rotary_frequencies
    g = _gen(6)
    q = _randn(g, 2, 9, 3, 16)
    pos = torch.randint(1_000_000, 16_000_000, (2, 9, 2), generator=g).to(DEV).to(ptype)
    if ptype.is_floating_point:
        pos = pos / 8 + 0.5
    f = rotary_frequencies((5, 3), device=DEV)
    oq, ok = rotary_axes(q, None, pos, f, (5, 3))
    assert ok is None
    mag = q.abs().double() + torch.cat([q[..., 8:], q[..., :8]], -1).abs().double()
    _within(oq, ref.rotary(q, pos, f, (5, 3)), 13 * 2.0 ** -24 * mag, "q")


def test_rotary_strides_shared_positions_and_one_gradient():
    """q and k as views of one projection, positions shared over the batch, only one input's gradient."""
    from sldm_sage import rotary_axes, rotary_frequencies
    g = _gen(7)
    both = _randn(g, 3, 11, 9, 24, dtype=torch.bfloat16)
    q, k = both[:, :, :6, 1:21], both[:, :, 6:, 1:21]          # rows start off 16-byte boundaries
    pos = torch.arange(11, device=DEV)[None, :, None].expand(3, 11, 2)
    f = rotary_frequencies((4, 6), device=DEV)
    oq, ok = rotary_axes(q, k, pos, f, (4, 6), interleaved=True)
    for got, x in ((oq, q), (ok, k)):
        c = x.contiguous()
        again, _ = rotary_axes(c, None, pos.contiguous(), f, (4, 6), interleaved=True)
        assert torch.equal(got, again)
    x = _randn(g, 3, 11, 3, 24)
    leaf = x.clone().requires_grad_(True)
    first, second = rotary_axes(x, leaf, pos, f, (4, 6))
    assert second.requires_grad
    gk = _randn(g, 3, 11, 3, 24)
    d, = torch.autograd.grad(second, leaf, gk)
    back, _ = rotary_axes(gk, None, -pos, f, (4, 6))
    _within(d, back.double(), 2.0 ** -22 * gk.abs().double().amax(), "dk")
    t = x.transpose(2, 3).contiguous().transpose(2, 3)         # columns not contiguous
    assert torch.equal(rotary_axes(t, None, pos, f, (4, 6))[0], first)


# ---------------------------------------------------------- decay attention --
def _decays(h, kind="mixed"):
    if kind == "mixed":
        return torch.log1p(-torch.exp2(-1.0 - torch.arange(h) * 6.0 / max(h, 1))).to(DEV)
    return torch.full((h,), {"none": 0.0, "strong": -30.0, "all": -math.inf}[kind], device=DEV)


def _att_bounds(u, T, out, mag):
    """bf16 also rounds Q K^T o D (u mag) and reads the state as hi + lo (2^-16 mag)."""
    extra = u + 2.0 ** -16 if u > 2.0 ** -20 else 0.0
    return u * out.abs() + (extra + (T + 256) * 2.0 ** -24) * mag


def _check_attention(q, k, v, ld, scale, state, lengths, do, dend, dtype):
    from sldm_sage import decay_attention
    T = q.size(1)
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, v, state)]
    o, end = decay_attention(leaves[0], leaves[1], leaves[2], ld, scale=scale, state=leaves[3], lengths=lengths)
    assert o.dtype == dtype and end.dtype == torch.float32
    inputs = [t for t in leaves if t is not None]
    grads = torch.autograd.grad((o, end), inputs, (do, dend))
    scale = q.size(-1) ** -0.5 if scale is None else scale
    lens = lengths
    keep = torch.ones(q.shape[:2], dtype=torch.bool, device=DEV) if lens is None else \
        torch.arange(T, device=DEV) < lens[:, None]
    m = keep[..., None, None]

    def clean(t):    # what padding holds does not count
        return torch.where(m, t, torch.zeros_like(t))
    args = [clean(t) for t in (q, k, v)]
    (wo, wend), wg = ref.decay_attention(*args, ld, scale, state, lens, clean(do), dend)
    (mo, mend), mg = ref.decay_attention(*(t.abs() for t in args), ld, abs(scale),
                                         None if state is None else state.abs(), lens, clean(do).abs(), dend.abs())
    u = U[dtype]
    _within(o, wo, _att_bounds(u, T, wo, mo), "out")
    _within(end, wend, _att_bounds(2.0 ** -24, T, wend, mend), "state")
    for name, got, want, mag, uu in zip(("dq", "dk", "dv", "dstate"), grads, wg, mg, (u, u, u, 2.0 ** -24)):
        _within(got, want, _att_bounds(uu, T, want, mag), name)
    if lens is not None:
        for t in (o, *grads[:3]):
            assert not t[~keep].any()
    return o, end, grads


ATTENTION = [  # B, T, H, Hk, Dk, Dv
    (1, 1, 1, 1, 1, 1), (2, 2, 1, 1, 16, 16), (1, 31, 2, 2, 32, 32), (2, 32, 2, 2, 16, 32), (2, 33, 3, 3, 24, 8),
    (3, 63, 2, 1, 64, 64), (2, 64, 2, 2, 64, 32), (2, 65, 4, 2, 40, 72), (5, 100, 6, 6, 16, 16), (1, 129, 2, 2, 128, 128),
    (2, 130, 4, 1, 48, 80), (1, 200, 2, 2, 128, 24), (1, 257, 1, 1, 20, 128), (2, 97, 2, 2, 33, 7), (3, 70, 2, 2, 96, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_state", [False, True], ids=["zeros", "state"])
@pytest.mark.parametrize("case", ATTENTION, ids=str)
def test_decay_attention(case, with_state, dtype):
    B, T, H, Hk, Dk, Dv = case
    g = _gen(8)
    q, k, v = (_randn(g, B, T, h, d, dtype=dtype) for h, d in ((H, Dk), (Hk, Dk), (Hk, Dv)))
    do, dend = _randn(g, B, T, H, Dv, dtype=dtype), _randn(g, B, H, Dk, Dv)
    state = _randn(g, B, H, Dk, Dv) if with_state else None
    _check_attention(q, k, v, _decays(H), None, state, None, do, dend, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["none", "strong", "all"])
def test_decay_attention_decay_extremes(kind, dtype):
    """No decay (a plain sum), one that keeps e^-30 a token, and -inf (each token alone)."""
    g = _gen(9)
    q, k, v, do = (_randn(g, 2, 150, 2, 32, dtype=dtype) for _ in range(4))
    state, dend = _randn(g, 2, 2, 32, 32), _randn(g, 2, 2, 32, 32)
    lengths = torch.tensor([150, 0], dtype=torch.int32, device=DEV)
    _check_attention(q, k, v, _decays(2, kind), 0.5, state, lengths, do, dend, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
@pytest.mark.parametrize("heads", [(2, 1, 32, 48), (6, 6, 16, 16)], ids=str)
@pytest.mark.parametrize("T", [5, 70, 300, 700])
def test_decay_attention_ragged(T, heads, itype, dtype):
    """Lengths 0, 1, at and around the chunks' ends, beyond T and below 0 (clamped); NaN and Inf behind them."""
    g = _gen(10)
    lens = torch.tensor([0, 1, T, T + 9, -3, min(T, 31), min(T, 64), min(T, 65), T - 1, T // 2], dtype=itype, device=DEV)
    B, (H, Hk, Dk, Dv) = lens.numel(), heads
    q, k, v = (_randn(g, B, T, h, d, dtype=dtype) for h, d in ((H, Dk), (Hk, Dk), (Hk, Dv)))
    do, dend, state = _randn(g, B, T, H, Dv, dtype=dtype), _randn(g, B, H, Dk, Dv), _randn(g, B, H, Dk, Dv)
    behind = ~(torch.arange(T, device=DEV) < lens[:, None])
    for n, t in enumerate((q, k, v, do)):
        t[behind] = (float("nan"), float("inf"), -float("inf"), float("nan"))[n]
    o, end, grads = _check_attention(q, k, v, _decays(H), None, state, lens, do, dend, dtype)
    assert torch.equal(end[0], state[0]) and torch.equal(grads[3][0], dend[0])     # no token: the state as it was


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(1, 2500, 2, 1, 64, 64), (2, 1111, 1, 1, 128, 40), (1, 4100, 1, 1, 16, 16),
                                  (2, 2100, 4, 4, 16, 16)], ids=str)
def test_decay_attention_long_axis(case, dtype):
    """Few heads and a long axis: the axis is cut into segments."""
    B, T, H, Hk, Dk, Dv = case
    g = _gen(11)
    q, k, v = (_randn(g, B, T, h, d, dtype=dtype) for h, d in ((H, Dk), (Hk, Dk), (Hk, Dv)))
    do, dend, state = _randn(g, B, T, H, Dv, dtype=dtype), _randn(g, B, H, Dk, Dv), _randn(g, B, H, Dk, Dv)
    lens = None if B == 1 else torch.tensor([T, T // 3], device=DEV)
    ld = torch.log1p(-torch.exp2(-4.0 - 3 * torch.arange(H))).to(DEV)
    _check_attention(q, k, v, ld, None, state, lens, do, dend, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "do", "state"])
@pytest.mark.parametrize("case", [(3, 70, 2, 1, 32, 48), (2, 45, 2, 2, 33, 7), (1, 1500, 1, 1, 64, 64), (2, 97, 4, 2, 128, 100),
                                  (1, 700, 1, 1, 16, 16), (2, 75, 4, 4, 16, 16)], ids=str)
def test_decay_attention_infinities_and_nan_stay_causal(case, which, dtype):
    """One value that is not finite, in the middle of a chunk, reaches what the recurrences say and nothing else:
    no output of an earlier token (of a later one, for the gradients of k and v), no other column of v."""
    from sldm_sage import decay_attention
    B, T, H, Hk, Dk, Dv = case
    g = _gen(31)
    t = {"q": _randn(g, B, T, H, Dk, dtype=dtype), "k": _randn(g, B, T, Hk, Dk, dtype=dtype),
         "v": _randn(g, B, T, Hk, Dv, dtype=dtype), "do": _randn(g, B, T, H, Dv, dtype=dtype),
         "state": _randn(g, B, H, Dk, Dv)}
    dend, ld, scale = _randn(g, B, H, Dk, Dv), _decays(H), Dk ** -0.5
    hit = t[which]
    if which == "state":
        hit[0, 0, Dk // 2, Dv // 3] = float("inf")
    else:
        hit[0, T // 2 + 3, 0, hit.size(3) // 2] = float("nan" if which in "qv" else "inf")
        hit[0, T - 2, -1, 0] = -float("inf")
    leaves = [t[n].clone().requires_grad_(True) for n in ("q", "k", "v", "state")]
    o, end = decay_attention(*leaves[:3], ld, state=leaves[3])
    grads = torch.autograd.grad((o, end), leaves, (t["do"], dend))
    (wo, wend), wg = ref.decay_attention(t["q"], t["k"], t["v"], ld, scale, t["state"], None, t["do"], dend)
    a = {n: x.abs() for n, x in t.items()}
    (mo, mend), mg = ref.decay_attention(a["q"], a["k"], a["v"], ld, scale, a["state"], None, a["do"], dend.abs())
    u, e = U[dtype], U[torch.float32]
    some = False
    for name, got, want, mag, uu in zip(("out", "state", "dq", "dk", "dv", "dstate"), (o, end, *grads), (wo, wend, *wg),
                                        (mo, mend, *mg), (u, e, u, u, u, e)):
        fine = want.isfinite()
        some |= not fine.all()
        assert torch.equal(got.isfinite(), fine), name
        _within(got[fine], want[fine], _att_bounds(uu, T, want, mag)[fine], name)
    assert some


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_attention_strides(dtype):
    """Views of one projection, head-major tensors, expanded heads and gradients, columns not contiguous."""
    from sldm_sage import decay_attention
    g = _gen(12)
    B, T, H, D = 2, 77, 3, 32
    ld = _decays(H)
    packed = _randn(g, B, T, 3 * H * D + 5, dtype=dtype)
    q, k, v = packed[..., 5:].unflatten(-1, (3, H, D)).unbind(2)               # off 16-byte boundaries
    a = decay_attention(q, k, v, ld)
    b = decay_attention(q.contiguous(), k.contiguous(), v.contiguous(), ld)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    hm = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    c = decay_attention(*hm, ld)
    assert torch.equal(c[0], b[0]) and torch.equal(c[1], b[1])
    cm = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    c = decay_attention(*cm, ld)
    assert torch.equal(c[0], b[0])
    one = q[:, :, :1].expand(B, T, H, D)
    leaf = one.detach().requires_grad_(True)
    o, _ = decay_attention(leaf, k, v, ld)
    do = _randn(g, D, dtype=dtype).expand(B, T, H, D)
    d1, = torch.autograd.grad(o, leaf, do)
    leaf2 = one.contiguous().requires_grad_(True)
    d2, = torch.autograd.grad(decay_attention(leaf2, k, v, ld)[0], leaf2, do.contiguous())
    assert torch.equal(d1, d2)


def test_decay_attention_one_long_dimension_strides():
    """Dimensions of one with strides that mean nothing; one token of a long cache; time-major tensors."""
    from sldm_sage import decay_attention
    g = _gen(21)
    x = _randn(g, 3, 50, 5, 16, dtype=torch.bfloat16)
    ld = _decays(1)
    one = x[1:2, :, 2:3].as_strided((1, 50, 1, 16), (7, x.stride(1), 3, 1), x[1:2, :, 2:3].storage_offset())
    a, b = decay_attention(one, one, one, ld), decay_attention(*(x[1:2, :, 2:3].contiguous(),) * 3, ld)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    tm = _randn(g, 60, 4, 2, 16)                                    # [T, B, H, D]
    a = decay_attention(*(tm.transpose(0, 1),) * 3, _decays(2))
    b = decay_attention(*(tm.transpose(0, 1).contiguous(),) * 3, _decays(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_attention_offsets_beyond_32_bits(dtype):
    """Sequences whose bytes lie beyond 2^32 of the tensor's start (an expanded view costs no such memory to
    read, a token stride beyond the fast path's reach takes the slow one)."""
    from sldm_sage import decay_attention
    g = _gen(22)
    n = (1 << 32) // torch.empty(0, dtype=dtype).element_size() + 4096
    big = torch.zeros(n, dtype=dtype, device=DEV)
    small = _randn(g, 1, 40, 2, 16, dtype=dtype)
    ld = _decays(2)
    want = decay_attention(small, small, small, ld)
    far = big[-40 * 32:].view(1, 40, 2, 16)
    far.copy_(small)
    batch = big.as_strided((2, 40, 2, 16), (n - 40 * 32, 32, 16, 1))     # batch 1 is `far`
    o, s = decay_attention(batch, batch, batch, ld)
    assert torch.equal(o[1], want[0][0]) and torch.equal(s[1], want[1][0]) and not o[0].any()
    step = (n - 32) // 39                                               # tokens far apart
    step -= step % 8
    wide = big.as_strided((1, 40, 2, 16), (0, step, 16, 1))
    wide.copy_(small)
    o, s = decay_attention(wide, wide, wide, ld)
    (wo, ws), (mo, ms) = (ref.decay_attention(t, t, t, ld, 0.25) for t in (small, small.abs()))
    _within(o, wo, _att_bounds(U[dtype], 40, wo, mo), "out")
    _within(s, ws, _att_bounds(2.0 ** -24, 40, ws, ms), "state")


def test_second_derivatives_are_refused():
    from sldm_sage import decay_attention, layer_norm, rotary_axes, rotary_frequencies
    x = torch.randn(2, 5, 2, 16, device=DEV, requires_grad=True)
    pos, f = torch.zeros(2, 5, 1, device=DEV), rotary_frequencies((8,), device=DEV)
    for y in (layer_norm(x), rotary_axes(x, None, pos, f, (8,))[0], decay_attention(x, x, x, _decays(2))[0]):
        with pytest.raises(RuntimeError, match="cannot be differentiated"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.parametrize("T", [90, 1300])
def test_decay_attention_single_gradients(T):
    """Each gradient alone, and with only one of the two outputs used, equals that of the whole."""
    from sldm_sage import decay_attention
    g = _gen(13)
    q, k, v = (_randn(g, 1, T, h, 32).requires_grad_(True) for h in (2, 1, 1))
    state = _randn(g, 1, 2, 32, 32).requires_grad_(True)
    ld = _decays(2)
    do, dend = _randn(g, 1, T, 2, 32), _randn(g, 1, 2, 32, 32)
    out = decay_attention(q, k, v, ld, state=state)
    whole = torch.autograd.grad(out, (q, k, v, state), (do, dend), retain_graph=True)
    for t, w in zip((q, k, v, state), whole):
        assert torch.equal(torch.autograd.grad(out, t, (do, dend), retain_graph=True)[0], w)
    from_o = torch.autograd.grad(out[0], (q, k, v, state), do, retain_graph=True)
    from_s = torch.autograd.grad(out[1], (q, k, v, state), dend, allow_unused=True)
    (_, _), wo = ref.decay_attention(q.detach(), k.detach(), v.detach(), ld, 32 ** -0.5, state.detach(), None, do,
                                     torch.zeros_like(dend))
    (_, _), ws = ref.decay_attention(q.detach(), k.detach(), v.detach(), ld, 32 ** -0.5, state.detach(), None,
                                     torch.zeros_like(do), dend)
    (_, _), mag = ref.decay_attention(q.detach().abs(), k.detach().abs(), v.detach().abs(), ld, 32 ** -0.5,
                                      state.detach().abs(), None, do.abs(), dend.abs())
    for name, a, b, wa, wb, m in zip("qkvs", from_o, from_s, wo, ws, mag):
        _within(a, wa, _att_bounds(2.0 ** -24, T, wa, m), "d" + name + " of out")
        _within(b, wb, _att_bounds(2.0 ** -24, T, wb, m), "d" + name + " of state")


def test_decay_attention_gradient_against_differences():
    """out and state are linear in each of q, k, v and the first state: a difference over a whole step is
    the directional derivative, up to the rounding of both evaluations."""
    from sldm_sage import decay_attention
    g = _gen(14)
    B, T, H, D = 2, 75, 2, 24
    base = [_randn(g, B, T, H, D) for _ in range(3)] + [_randn(g, B, H, D, D)]
    ld, do, dend = _decays(H), _randn(g, B, T, H, D), _randn(g, B, H, D, D)

    def loss(t):
        o, s = decay_attention(t[0], t[1], t[2], ld, state=t[3])
        return (o.double() * do).sum() + (s.double() * dend).sum()
    leaves = [t.clone().requires_grad_(True) for t in base]
    o, s = decay_attention(leaves[0], leaves[1], leaves[2], ld, state=leaves[3])
    grads = torch.autograd.grad((o, s), leaves, (do, dend))
    for n in range(4):
        step = _randn(g, *base[n].shape)
        up, down = list(base), list(base)
        up[n], down[n] = base[n] + step, base[n] - step
        diff = (loss(up) - loss(down)) / 2
        dot = (grads[n].double() * step.double()).sum()
        mags = [t.abs() for t in base]
        mags[n] = base[n].abs() + step.abs()
        (mo, ms), _ = ref.decay_attention(*mags[:3], ld, D ** -0.5, mags[3], None, do.abs(), dend.abs())
        mag = (mo * do.abs()).sum() + (ms * dend.abs()).sum()
        assert abs(float(diff - dot)) <= 2 * (T + 256) * 2.0 ** -24 * float(mag), (n, float(diff), float(dot))


def test_decay_attention_empty():
    from sldm_sage import decay_attention, decay_attention_step
    ld = _decays(2)
    for B, T in ((0, 5), (3, 0), (0, 0)):
        q = torch.empty(B, T, 2, 8, device=DEV, requires_grad=True)
        state = torch.randn(B, 2, 8, 8, device=DEV, requires_grad=True)
        o, s = decay_attention(q, q, q, ld, state=state)
        assert o.shape == (B, T, 2, 8) and torch.equal(s, state)
        gs = torch.ones_like(s)
        dq, ds = torch.autograd.grad((o, s), (q, state), (torch.ones_like(o), gs))
        assert dq.shape == q.shape and torch.equal(ds, gs)
        assert not decay_attention(q.detach(), q.detach(), q.detach(), ld)[1].any()
    e = torch.empty(0, 2, 8, device=DEV)
    assert decay_attention_step(e, e, e, ld, torch.empty(0, 2, 8, 8, device=DEV)).shape == (0, 2, 8)


# --------------------------------------------------------------------- step --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(1, 1, 1, 1, 1), (3, 6, 6, 16, 16), (2, 4, 2, 64, 64), (5, 2, 1, 128, 128),
                                  (2, 2, 2, 33, 7), (2, 3, 3, 40, 96), (4, 2, 2, 128, 4)], ids=str)
def test_decay_attention_step(case, dtype):
    from sldm_sage import decay_attention_step
    B, H, Hk, Dk, Dv = case
    g = _gen(15)
    ld = _decays(H)
    packed = _randn(g, B, H * Dk + Hk * (Dk + Dv), dtype=dtype)
    q, k, v = packed.split([H * Dk, Hk * Dk, Hk * Dv], -1)
    q, k, v = q.unflatten(-1, (H, Dk)), k.unflatten(-1, (Hk, Dk)), v.unflatten(-1, (Hk, Dv))
    state = _randn(g, B, H, Dk, Dv)
    s = state.clone()
    version = s._version
    o = decay_attention_step(q, k, v, ld, s)
    assert s._version > version
    args = [t.unsqueeze(1) for t in (q, k, v)]
    wo, ws = ref.decay_attention(*args, ld, Dk ** -0.5, state)
    mo, ms = ref.decay_attention(*(t.abs() for t in args), ld, Dk ** -0.5, state.abs())
    _within(s, ws, 4 * 2.0 ** -24 * ms, "state")            # a product, a sum, g
    _within(o, wo[:, 0], U[dtype] * wo[:, 0].abs() + (Dk + 8) * 2.0 ** -24 * mo[:, 0], "out")


@pytest.mark.parametrize("dtype", DTYPES)
def test_decay_attention_goes_on(dtype):
    """A sequence in one call, in pieces that hand the state on, and token by token."""
    from sldm_sage import decay_attention, decay_attention_step
    g = _gen(16)
    B, T, H, D = 3, 90, 2, 32
    q, k, v = (_randn(g, B, T, H, D, dtype=dtype) for _ in range(3))
    ld = _decays(H)
    (wo, ws), (mo, ms) = (ref.decay_attention(*a, ld, D ** -0.5) for a in ((q, k, v), (q.abs(), k.abs(), v.abs())))
    bound_o, bound_s = _att_bounds(U[dtype], T, wo, mo), _att_bounds(2.0 ** -24, T, ws, ms)
    state, outs, at = None, [], 0
    for n in (1, 40, 3, 46):
        o, state = decay_attention(q[:, at:at + n], k[:, at:at + n], v[:, at:at + n], ld, state=state)
        outs.append(o)
        at += n
    _within(torch.cat(outs, 1), wo, bound_o, "pieces")
    _within(state, ws, bound_s, "state of pieces")
    state = torch.zeros(B, H, D, D, device=DEV)
    outs = [decay_attention_step(q[:, t], k[:, t], v[:, t], ld, state) for t in range(T)]
    _within(torch.stack(outs, 1), wo, bound_o, "steps")
    _within(state, ws, bound_s, "state of steps")


# ------------------------------------------------- streams, graphs, the whole --
def test_sequence_ops_deterministic_and_on_another_stream():
    from sldm_sage import decay_attention, layer_norm, rotary_axes, rotary_frequencies
    g = _gen(17)
    x0 = _randn(g, 4, 700, 2, 32)
    pos = torch.arange(700, device=DEV)[None, :, None].expand(4, 700, 1)
    f, ld = rotary_frequencies((16,), device=DEV), _decays(2)

    def run():
        x, w = x0.clone().requires_grad_(True), torch.ones(32, device=DEV, requires_grad=True)
        h = layer_norm(x, w)
        q, k = rotary_axes(h, h, pos, f, (16,))
        o, s = decay_attention(q, k, h, ld)
        return (o.detach(), s.detach(), *torch.autograd.grad((o.sum() + s.sum()), (x, w)))
    first = run()
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))


@pytest.mark.parametrize("T", [80, 1500])
def test_sequence_ops_under_capture(T):
    """A forward and backward pass recorded into a graph, replayed on new inputs, equals the eager one; two
    graphs of different shapes replay in turn."""
    from sldm_sage import decay_attention, layer_norm, rotary_axes, rotary_frequencies
    g = _gen(18)
    f, ld = rotary_frequencies((16,), device=DEV), _decays(4)

    def program(x, w, pos, lens):
        h = layer_norm(x, w)
        q, k = rotary_axes(h, h[:, :, :2], pos, f, (16,))
        o, s = decay_attention(q, k, h[:, :, 2:], ld, lengths=lens)
        return (o, s, *torch.autograd.grad((o, s), (x, w), (torch.ones_like(o), torch.ones_like(s))))

    def buffers(t):
        return (torch.zeros(1, t, 4, 32, device=DEV), torch.ones(32, device=DEV),
                torch.zeros(1, t, 1, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    graphs = []
    for t in (T, T // 2 + 1):
        bufs = buffers(t)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            program(*(b.detach().requires_grad_(b.is_floating_point()) for b in bufs))
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = program(*(b.detach().requires_grad_(b.is_floating_point()) for b in bufs))
        graphs.append((t, bufs, graph, outs))
    for turn in range(3):
        for t, bufs, graph, outs in graphs:
            x = _randn(g, 1, t, 4, 32)
            pos = torch.randint(0, 5000, (1, t, 1), generator=g).to(DEV)
            lens = torch.tensor([t - 3 * turn], dtype=torch.int32, device=DEV)
            for b, new in zip(bufs, (x, 1 + 0.1 * _randn(g, 32), pos, lens)):
                b.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            want = program(*(b.clone().requires_grad_(b.is_floating_point()) for b in bufs))
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_decay_encoder_runs_like_the_gru():
    """The encoder: one call, pieces that hand the state on, live frames, gradients of every parameter."""
    from sldm_sage import DecayEncoder
    torch.manual_seed(0)
    enc = DecayEncoder(6, 96, num_heads=6, sections=(2, 3, 3)).to(DEV)
    x = torch.randn(7, 40, 6, device=DEV)
    pos = torch.cat([torch.arange(40, device=DEV)[None, :, None].expand(7, 40, 1).float(),
                     torch.randn(7, 40, 2, device=DEV) * 30], -1)
    lens = torch.tensor([40, 3, 17, 0, 40, 1, 33], device=DEV)
    out, (S, seen) = enc(x, positions=pos, lengths=lens)
    assert out.shape == (7, 40, 96) and torch.equal(seen, lens)
    (out.square().mean() + S.square().mean()).backward()
    for name, p in enc.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all() and p.grad.abs().sum() > 0, name
    with torch.no_grad():
        whole, end = enc(x, positions=pos)
        a, state = enc(x[:, :25], positions=pos[:, :25])
        b, state = enc(x[:, 25:], state, positions=pos[:, 25:])
        # the same sums in other chunks: fp32 rounding through two norms and a projection
        torch.testing.assert_close(torch.cat([a, b], 1), whole, atol=1e-4, rtol=1e-4)
        live = enc.init_state(7, device=DEV)
        frames = [enc.step(x[:, t], live, pos[:, t]) for t in range(40)]
        torch.testing.assert_close(torch.stack(frames, 1), whole, atol=1e-4, rtol=1e-4)
        assert torch.equal(live[1], end[1])
    # against the same encoder written with the oracle in 64 bits
    with torch.no_grad():
        d = {k: v.double() for k, v in enc.state_dict().items()}
        h = torch.nn.functional.silu(x.double() @ d["embed.weight"].T + d["embed.bias"])
        n = ref.layer_norm(h, d["norm.weight"], d["norm.bias"])
        q, k, v = (n @ d["qkv.weight"].T).unflatten(-1, (3, 6, 16)).unbind(-3)
        f = enc._inv_freq.to(DEV)
        q, k = ref.rotary(q, pos, f, enc.sections), ref.rotary(k, pos, f, enc.sections)
        o, _ = ref.decay_attention(q, k, v, enc._log_decay.to(DEV), 0.25)
        want = h + ref.layer_norm(o).flatten(-2) @ d["proj.weight"].T
        torch.testing.assert_close(whole.double(), want, atol=1e-4, rtol=1e-4)


def test_decay_encoder_served_before_it_is_trained():
    """The first call under inference_mode leaves nothing behind that a training pass cannot save."""
    from sldm_sage import DecayEncoder
    torch.manual_seed(1)
    enc = DecayEncoder(6, 64, num_heads=2).to(DEV)
    x = torch.randn(3, 9, 6, device=DEV)
    with torch.inference_mode():
        served, _ = enc(x)
        live = enc.init_state(3)
        frames = torch.stack([enc.step(x[:, t], live) for t in range(9)], 1)
        torch.testing.assert_close(frames, served, atol=1e-4, rtol=1e-4)
    out, _ = enc(x)
    assert torch.equal(out.detach(), served)
    out.sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in enc.parameters())


def test_layer_norm_and_rotary_beyond_32_bits():
    """More than 2^31 elements, and rows further apart than that: the last rows equal the same rows alone."""
    from sldm_sage import layer_norm, rotary_axes, rotary_frequencies
    w = torch.linspace(0.5, 1.5, 256, device=DEV)
    x = torch.randn(8_400_000, 256, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    assert x.numel() > 2 ** 31
    y = layer_norm(x, w)
    dx, = torch.autograd.grad(y, x, x.detach())
    few = x.detach()[-1000:].clone().requires_grad_(True)
    z = layer_norm(few, w)
    assert torch.equal(y[-1000:], z)
    assert torch.equal(dx[-1000:], torch.autograd.grad(z, few, few.detach())[0])
    del y, dx, z
    wide = x.detach().view(-1)[:2 ** 31].view(2, 2 ** 30)[:, -256:]
    assert torch.equal(layer_norm(wide, w), layer_norm(wide.clone(), w))
    del x, wide
    T = 17_000_000
    q = torch.randn(T, 2, 64, device=DEV, dtype=torch.bfloat16)
    assert q.numel() > 2 ** 31
    f, pos = rotary_frequencies((20, 12), device=DEV), torch.arange(T, device=DEV)[:, None].expand(T, 2)
    out, _ = rotary_axes(q, None, pos, f, (20, 12))
    assert torch.equal(out[-1000:], rotary_axes(q[-1000:], None, pos[-1000:], f, (20, 12))[0])


def test_sequence_ops_from_two_host_threads():
    """Two threads, each on a stream of its own, at once: the results of one after the other."""
    import threading
    from sldm_sage import decay_attention, layer_norm, rotary_axes, rotary_frequencies
    g = _gen(41)
    f, ld = rotary_frequencies((8, 8), device=DEV), _decays(4)
    data = [(_randn(g, 2, t, 4, 32), torch.randint(0, 900, (2, t, 2), generator=g).to(DEV)) for t in (1300, 77)]

    def program(x, pos):
        leaf = x.clone().requires_grad_(True)
        h = layer_norm(leaf)
        q, k = rotary_axes(h, h[:, :, :2], pos, f, (8, 8))
        o, s = decay_attention(q, k, h[:, :, 2:], ld)
        return (o, s, *torch.autograd.grad((o, s), leaf, (torch.ones_like(o), torch.ones_like(s))))
    want = [program(*d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = program(*data[i])
            stream.synchronize()
        except Exception as e:      # reported below: a thread's own error would pass unseen
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_decay_encoder_under_capture():
    """A sequence, and live frames that move the state on in place, recorded and replayed on new inputs."""
    from sldm_sage import DecayEncoder
    torch.manual_seed(3)
    enc = DecayEncoder(6, 96, num_heads=6, sections=(2, 3, 3)).to(DEV).requires_grad_(False)
    x, pos = torch.zeros(5, 40, 6, device=DEV), torch.zeros(5, 40, 3, device=DEV)
    lens = torch.full((5,), 40, device=DEV)
    live = enc.init_state(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        enc(x, positions=pos, lengths=lens)
        enc.step(x[:, 0], live, pos[:, 0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    whole, one = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(whole):
        out, (S, seen) = enc(x, positions=pos, lengths=lens)
    with torch.cuda.graph(one):
        frame = enc.step(x[:, 0], live, pos[:, 0])
    for turn in range(3):
        x.copy_(torch.randn(5, 40, 6, device=DEV))
        pos.copy_(torch.randn(5, 40, 3, device=DEV) * 20)
        lens.copy_(torch.tensor([40, 0, 3 + turn, 32, 33], device=DEV))
        for t in live:
            t.zero_()
        whole.replay()
        torch.cuda.synchronize()
        want, (wS, wseen) = enc(x, positions=pos, lengths=lens)
        assert torch.equal(out, want) and torch.equal(S, wS) and torch.equal(seen, wseen)
        again = enc.init_state(5)
        for _ in range(4):
            one.replay()
            torch.cuda.synchronize()
            assert torch.equal(frame, enc.step(x[:, 0], again, pos[:, 0]))
        assert torch.equal(live[0], again[0]) and torch.equal(live[1], again[1])
