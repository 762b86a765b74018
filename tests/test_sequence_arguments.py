"""Calls of the sequence operators that have no answer and are refused; no kernel runs (CPU tensors)."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import sldm_sage as sage


def test_forward_mode_derivatives_are_refused():
    """A tangent would be dropped without a word, and read as a derivative of zero."""
    x, w = torch.randn(3, 8), torch.ones(8)
    q, pos, f = torch.zeros(2, 5, 2, 16), torch.zeros(2, 5, 1), sage.rotary_frequencies((8,))
    ld, state = torch.zeros(2), torch.zeros(2, 2, 16, 16)
    calls = [(sage.layer_norm, (x, w, w)), (sage.rotary_axes, (q, q, pos, f, (8,))),
             (lambda q, k, v, ld, s: sage.decay_attention(q, k, v, ld, state=s), (q, q, q, ld, state)),
             (sage.decay_attention_step, (q[:, 0], q[:, 0], q[:, 0], ld, state))]
    for call, args in calls:
        for i, a in enumerate(args):
            if not isinstance(a, torch.Tensor):
                continue
            for leaf in (False, True):
                with forward_ad.dual_level():
                    dual = forward_ad.make_dual(a.detach().clone(), torch.ones_like(a))
                    if leaf:
                        dual.requires_grad_(True)
                    with pytest.raises(RuntimeError, match="forward-mode|no gradient"), torch.set_grad_enabled(leaf):
                        call(*args[:i], dual, *args[i + 1:])
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no CPU fallback"):
                call(*args)                            # no tangent: on to the next check


def test_encoder_state_and_frame_are_checked():
    enc = sage.DecayEncoder(6, 96, num_heads=6)
    S, seen = enc.init_state(3)
    frame, frames = torch.zeros(3, 6), torch.zeros(3, 4, 6)
    for x in (torch.zeros(3, 7), torch.zeros(6), frames):
        with pytest.raises(ValueError, match=r"expected \[N, 6\]"):
            enc.step(x, (S, seen))
    for state in (S, None, (S,), (S, seen, seen), (S[:2], seen), (S, seen[:2]), (S, seen[:, None]), (S[..., :8], seen),
                  (S, 3), (seen, S)):
        with pytest.raises(ValueError, match="state is"):
            enc.step(frame, state)
        if state is not None:
            with pytest.raises(ValueError, match="state is"):
                enc(frames, state)
    for state in ((None, seen), (S, None)):
        with pytest.raises(ValueError, match="state is"):
            enc.step(frame, state)
    assert not seen.any() and not S.any()
    for call in (lambda: enc.step(frame, (S, seen)), lambda: enc(frames, (S, seen)), lambda: enc(frames, (S, None)),
                 lambda: enc(frames, (None, seen))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
