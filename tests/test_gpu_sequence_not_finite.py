"""Decay attention where values are not finite, or products leave fp32's range: an infinity or NaN reaches what the
recurrence says, with its kind and sign, and nothing else.  Bounds of the finite values: test_gpu_sequence_values.py."""
from __future__ import annotations

import pytest
import torch

from test_gpu_sequence import DEV, DTYPES, _decays, _gen, _randn
from test_gpu_sequence_values import NAMES, _both, _finite_within, _run

pytestmark = pytest.mark.gpu


def _same_kind(got, want, name):
    """NaN where the oracle has NaN, infinities where and of the sign that it has."""
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaN"
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf), f"{name}: infinities"
    assert torch.equal(got[inf].double().sign(), want[inf].sign()), f"{name}: signs"


# the tile classes, rows element by element, a cut axis (a segment's decay is 0 in fp32), pairs of narrow heads
KINDS = [(3, 70, 2, 1, 32, 48), (2, 45, 2, 2, 33, 7), (1, 1500, 1, 1, 64, 64), (2, 97, 4, 2, 128, 96),
         (1, 700, 1, 1, 16, 16), (2, 75, 4, 4, 16, 16)]


def _inputs(case, seed, dtype):
    B, T, H, Hk, Dk, Dv = case
    g = _gen(seed)
    return {"q": _randn(g, B, T, H, Dk, dtype=dtype), "k": _randn(g, B, T, Hk, Dk, dtype=dtype),
            "v": _randn(g, B, T, Hk, Dv, dtype=dtype), "do": _randn(g, B, T, H, Dv, dtype=dtype),
            "state": _randn(g, B, H, Dk, Dv), "dend": _randn(g, B, H, Dk, Dv)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")], ids=str)
@pytest.mark.parametrize("which", ["k", "v", "state"])
@pytest.mark.parametrize("case", KINDS, ids=str)
def test_the_state_keeps_an_infinity(case, which, value, dtype):
    """The returned state, and what goes on from it, holds the infinity that the recurrence holds."""
    from sldm_sage import decay_attention
    t, ld = _inputs(case, 61, dtype), _decays(case[2])
    at = (0, 0, 1, 2) if which == "state" else (0, case[1] // 2 + 3, 0, 2)
    t[which][at] = value
    args = (t["q"], t["k"], t["v"], ld, t["state"], None, t["do"], t["dend"])
    want, mag = _both(*args)
    o, end = decay_attention(*args[:4], state=t["state"])
    for name, a, w in (("out", o, want[0]), ("state", end, want[1])):
        _same_kind(a, w, name)
    _finite_within((o, end), want, mag, dtype, case[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["q", "k", "v", "do", "state", "dend"])
@pytest.mark.parametrize("case", KINDS, ids=str)
def test_kinds_and_signs(case, which, dtype):
    """Infinities of both signs and a NaN, inside a chunk: outputs, states and every gradient."""
    t, ld = _inputs(case, 62, dtype), _decays(case[2])
    B, T, hit = case[0], case[1], t[which]
    if which in ("state", "dend"):
        hit[0, -1, 3, 4], hit[-1, 0, 1, 0], hit[-1, 0, 5, 5] = float("inf"), -float("inf"), float("nan")
    else:
        hit[0, T // 2 + 3, -1, 3], hit[0, T - 2, 0, 5] = float("inf"), -float("inf")
        hit[-1, 7, 0, 1] = float("nan") if B > 1 else -float("inf")
    args = (t["q"], t["k"], t["v"], ld, t["state"], None, t["do"], t["dend"])
    got = _run(*args)
    want, mag = _both(*args)
    for name, a, w in zip(NAMES, got, want):
        _same_kind(a, w, name)
    _finite_within(got, want, mag, dtype, T)
    assert not all(w.isfinite().all() for w in want)


def _below_bf16(t, group):
    """What products below bf16's range may cost.  Inside a chunk an output is sum_j P_ij x_j with P_ij = q_i k_j
    times a decay <= 1 in two bf16 terms.  bf16's smallest step is 2^-133, so the terms are off by 2^-134 even
    where P is as small as that (here: do of 24 and v of 20, 1e-20 each), and the fp32 sum behind P, whose smallest
    step is 2^-149, by far less: together below 2^-133, times x_j, which is v (out), k (dq), q (dk) and do (dv),
    summed over the tokens, and over the heads that share a key head."""
    def up(x):
        return x.repeat_interleave(group, 2)

    def down(x):
        return x.unflatten(2, (-1, group)).sum(3)
    v, k, q, do = (2.0 ** -133 * t[n].double().abs().sum(1, keepdim=True) for n in ("v", "k", "q", "do"))
    return up(v), 0.0, up(k), down(q), down(do), 0.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(1, 40, 1, 1, 16, 16), (2, 40, 2, 2, 16, 16), (1, 70, 2, 1, 64, 128),
                                  (1, 45, 2, 2, 33, 7), (1, 1500, 1, 1, 64, 64)], ids=str)
def test_products_beyond_the_range_of_fp32(case, dtype):
    """q_i k_j of 1e50 where no entry of the recurrence is far out: of a later token j, which token i does not
    read (reversed in time for the gradients), and of an earlier one, whose v is small."""
    B, T, H, Hk, Dk, Dv = case
    t, ld = _inputs(case, 63, dtype), torch.full((H,), -0.01, device=DEV)
    t["state"].zero_()
    t["dend"].zero_()
    for first, second in ((3, 9), (T - 8, T - 2)):
        t["q"][:, first, :, 0] = 1e25          # token `first` does not read the key of `second`
        t["k"][:, second, :, 0] = 1e25
        t["v"][:, second] = 1e-20
        t["do"][:, first] = 1e-20
    t["k"][:, 20, :, 1] = 1e25                  # token 24 reads the key of 20
    t["v"][:, 20] = 1e-20
    t["q"][:, 24, :, 1] = 1e25
    t["do"][:, 24] = 1e-20
    args = (t["q"], t["k"], t["v"], ld, t["state"], None, t["do"], t["dend"])
    got = _run(*args)
    want, mag = _both(*args)
    for name, a, w in zip(NAMES, got, want):
        assert w.abs().max() < 1e38 and a.isfinite().all(), name
    _finite_within(got, want, mag, dtype, T, _below_bf16(t, H // Hk) if dtype == torch.bfloat16 else None)
