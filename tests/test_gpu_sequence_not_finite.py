"""Decay attention where values are not finite: an infinity or NaN reaches what the
recurrence says, with its kind and sign, and nothing else.  Bounds of the finite values: test_gpu_sequence_values.py."""
from __future__ import annotations

import pytest
import torch

from test_gpu_sequence import DTYPES, _decays, _gen, _randn
from test_gpu_sequence_values import _both, _finite_within

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
