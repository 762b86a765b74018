"""Decay attention where its roundings and its values that are not finite show (kernels: csrc/decay*.hip).

Against the recurrences in 64 bits (oracle/sequence_ref.py), elementwise.  The bound of a finite value: the
output's own rounding, u |out| with u = eps / 2 of its type (bf16 2^-8, fp32 2^-24); in bf16 an operand of a matrix
product that was fp32 goes in as two bf16 terms, each off by 2^-8 of what it rounds, together 2^-16 of the products'
magnitudes "mag" (the oracle's result for the magnitudes of the inputs); and the sums and weights of fp32,
(T + 256) 2^-24 mag as in test_gpu_sequence.py.
"""
from __future__ import annotations

import pytest
import torch

from oracle import sequence_ref as ref
from test_gpu_sequence import DEV, U, _decays, _gen, _randn, _within

pytestmark = pytest.mark.gpu
TWO_TERMS = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16}
NAMES = ("out", "state", "dq", "dk", "dv", "dstate")


def _bound(u, two, T, want, mag):
    return u * want.abs() + (two + (T + 256) * 2.0 ** -24) * mag


def _run(q, k, v, ld, state, lengths, do, dend):
    """out, state and the gradients of q, k, v (and the state), in the order of NAMES."""
    from sldm_sage import decay_attention
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, state) if t is not None]
    o, end = decay_attention(*leaves[:3], ld, state=None if state is None else leaves[3], lengths=lengths)
    return (o, end, *torch.autograd.grad((o, end), leaves, (do, dend)))


def _oracle(q, k, v, ld, state, lengths, do, dend):
    scale = q.size(-1) ** -0.5
    (o, end), g = ref.decay_attention(q, k, v, ld, scale, state, lengths, do, dend)
    return (o, end, *(g if state is not None else g[:3]))


def _both(q, k, v, ld, state, lengths, do, dend):
    args = (q, k, v, ld, state, lengths, do, dend)
    mags = (q.abs(), k.abs(), v.abs(), ld, None if state is None else state.abs(), lengths, do.abs(), dend.abs())
    return _oracle(*args), _oracle(*mags)


def _finite_within(got, want, mag, dtype, T, lost=None):
    """lost: what else each may be off by (None: nothing)."""
    for n, (name, a, w, m) in enumerate(zip(NAMES, got, want, mag)):
        fp32 = name in ("state", "dstate")
        u, two = (U[torch.float32], 0.0) if fp32 else (U[dtype], TWO_TERMS[dtype])
        fine = w.isfinite()
        bound = _bound(u, two, T, w, m) + (0.0 if lost is None else lost[n])
        _within(a[fine], w[fine], bound[fine], name)


# B, T, H, Hk, Dk, Dv: one chunk and some, whole walks, a cut axis (shared heads, wide heads), rows element by element
ROUNDINGS = [(2, 40, 2, 2, 16, 16), (2, 100, 2, 2, 64, 64), (2, 300, 3, 3, 32, 48), (3, 260, 2, 1, 96, 128),
             (1, 2500, 2, 1, 64, 64), (1, 1111, 1, 1, 128, 40), (2, 150, 2, 2, 33, 7)]


@pytest.mark.parametrize("with_state", [False, True], ids=["zeros", "state"])
@pytest.mark.parametrize("case", ROUNDINGS, ids=str)
def test_bf16_outputs_that_cancel(case, with_state):
    """Every output is the difference of two large entries of the state, so that a rounding of the state, or of
    the products inside a chunk, to bf16 shows in full: q and do have two columns, of opposite signs; k, v and the
    states are positive."""
    B, T, H, Hk, Dk, Dv = case
    g, bf = _gen(51), torch.bfloat16

    def positive(*shape, dtype=bf):
        return (_randn(g, *shape).abs() + 0.5).to(dtype)

    def two_columns(h, d):
        x = torch.zeros(B, T, h, d, dtype=bf, device=DEV)
        x[..., 0], x[..., d // 2 + 1] = positive(B, T, h), -positive(B, T, h)
        return x
    q, do = two_columns(H, Dk), two_columns(H, Dv)
    k, v, dend = positive(B, T, Hk, Dk), positive(B, T, Hk, Dv), torch.zeros(B, H, Dk, Dv, device=DEV)
    state = positive(B, H, Dk, Dv, dtype=torch.float32) if with_state else None
    ld = torch.log1p(-torch.exp2(-3.0 - 2 * torch.arange(H))).to(DEV)
    args = (q, k, v, ld, state, None, do, dend)
    got = _run(*args)
    want, mag = _both(*args)
    _finite_within(got, want, mag, bf, T)


@pytest.mark.parametrize("T", [100, 300, 2000])
def test_bf16_roundings_do_not_hang_on_the_state_being_given(T):
    """No state and a state of zeros are the same numbers."""
    g = _gen(52)
    q, k, v, do = (_randn(g, 2, T, 3, 32, dtype=torch.bfloat16) for _ in range(4))
    dend, ld = _randn(g, 2, 3, 32, 32), _decays(3)
    a = _run(q, k, v, ld, None, None, do, dend)
    b = _run(q, k, v, ld, torch.zeros(2, 3, 32, 32, device=DEV), None, do, dend)
    for name, x, y in zip(NAMES, a, b):
        assert torch.equal(x, y), name
