"""Decay attention on a cut time axis whose backward walks segments of their own: several of the forward's each, a
last one that is shorter, or none where only the forward is cut."""
from __future__ import annotations

import pytest
import torch

from test_gpu_sequence import DEV, DTYPES, _gen, _randn
from test_gpu_sequence_values import NAMES, _both, _finite_within, _run

pytestmark = pytest.mark.gpu


def _cut(dtype, B, T, H, Hk, Dk, Dv):
    """Segments of the forward (1: not cut), and whether the backward is cut, from what they ask room for."""
    from sldm_sage import _lib
    lib, code = _lib.load(), _lib.F32 if dtype == torch.float32 else _lib.BF16
    states = lib.sldm_decay_attention_states_bytes(code, B, T, H, Hk, Dk, Dv)
    parts = 0 if H == Hk else B * T * H * (Dk + Dv) * 4
    room = lib.sldm_decay_attention_bwd_workspace_bytes(code, B, T, H, Hk, Dk, Dv) - parts
    return max(1, states // (B * H * Dk * Dv * 4)), room > 0


def _check(case, dtype, ragged, with_state):
    B, T, H, Hk, Dk, Dv = case
    g = _gen(71)
    q, k, v = (_randn(g, B, T, h, d, dtype=dtype) for h, d in ((H, Dk), (Hk, Dk), (Hk, Dv)))
    do, dend = _randn(g, B, T, H, Dv, dtype=dtype), _randn(g, B, H, Dk, Dv)
    state = _randn(g, B, H, Dk, Dv) if with_state else None
    lens = torch.linspace(T, T // 5, B).long().to(DEV) if ragged else None
    if ragged:                                         # padding does not count, and comes out as zeros
        behind = ~(torch.arange(T, device=DEV) < lens[:, None])
        for t in (q, k, v, do):
            t[behind] = 0
    ld = torch.log1p(-torch.exp2(-3.0 - 7 * torch.arange(H) / H)).to(DEV)
    args = (q, k, v, ld, state, lens, do, dend)
    got = _run(*args)
    want, mag = _both(*args)
    _finite_within(got, want, mag, dtype, T)
    if ragged:
        for name, t in zip(NAMES, got):
            assert name.endswith("state") or not t[behind].any(), name


# heads enough that the waves, not the length, say how many segments there are: 15 of the forward's, two in each of
# the backward's, in bf16; 27 and 26, three in each, in fp32 (the counts of csrc/decay.hip: plans)
SEVERAL = [(4, 4200, 32, 32, 16, 16), (2, 4100, 64, 16, 16, 24)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ragged", [False, True], ids=["whole", "ragged"])
@pytest.mark.parametrize("case", SEVERAL, ids=str)
def test_several_forward_segments_in_one_of_the_backward(case, ragged, dtype):
    nseg, backward = _cut(dtype, *case)
    assert backward and nseg % (3 if dtype == torch.float32 and case[2] == 64 else 2), nseg
    _check(case, dtype, ragged, with_state=ragged)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", [(4, 1100, 128, 128, 16, 16), (8, 1100, 64, 32, 24, 16)], ids=str)
def test_only_the_forward_is_cut(case, dtype):
    nseg, backward = _cut(dtype, *case)
    assert nseg > 1 and not backward
    _check(case, dtype, True, with_state=True)
