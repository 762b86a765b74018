"""What the sequence operators refuse, with the message a user needs; no kernel runs (CPU tensors)."""
from __future__ import annotations

import pytest
import torch

import sldm_sage as sage


def _qkv(B=2, T=5, H=4, Hk=2, Dk=16, Dv=8, dtype=torch.float32):
    return torch.zeros(B, T, H, Dk, dtype=dtype), torch.zeros(B, T, Hk, Dk, dtype=dtype), \
        torch.zeros(B, T, Hk, Dv, dtype=dtype)


LD = torch.zeros(4)


def test_cpu_tensors_have_no_fallback():
    q, k, v = _qkv()
    f = sage.rotary_frequencies((8,))
    for call in (lambda: sage.layer_norm(torch.zeros(3, 4)),
                 lambda: sage.rotary_axes(q, k, torch.zeros(2, 5, 1), f, (8,)),
                 lambda: sage.decay_attention(q, k, v, LD),
                 lambda: sage.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], LD, torch.zeros(2, 4, 16, 8))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_layer_norm_refusals():
    x = torch.zeros(3, 8)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        sage.layer_norm(x.half())
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        sage.layer_norm(x.long())
    with pytest.raises(ValueError, match=r"weight and bias are \[8\]"):
        sage.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="weight and bias"):
        sage.layer_norm(x, torch.ones(8), torch.ones(1))
    with pytest.raises(TypeError, match="weight and bias"):
        sage.layer_norm(x, torch.ones(8).double())
    with pytest.raises(ValueError, match="last dimension"):
        sage.layer_norm(torch.zeros(()))
    with pytest.raises(ValueError, match="last dimension"):
        sage.layer_norm(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="eps"):
        sage.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="last dimension only"):
        sage.LayerNorm((3, 4))
    with pytest.raises(ValueError, match="expected"):
        sage.LayerNorm(8)(torch.zeros(2, 9))


def test_rotary_refusals():
    q, k, _ = _qkv()
    pos, f = torch.zeros(2, 5, 2), sage.rotary_frequencies((3, 5))

    def bad(err, match, q=q, k=k, pos=pos, f=f, sections=(3, 5)):
        with pytest.raises(err, match=match):
            sage.rotary_axes(q, k, pos, f, sections)
    bad(TypeError, "float32 or bfloat16", q=q.double())
    bad(TypeError, "rotary_axes: q is", k=k.bfloat16())
    bad(ValueError, "q is .*, k", k=k[:, :4])
    bad(ValueError, "q is .*, k", k=k[..., :8])
    bad(ValueError, "tokens, heads", q=q[0, 0], k=None)
    bad(ValueError, "positions are", pos=pos[..., :1])
    bad(ValueError, "positions are", pos=pos[:1])
    bad(TypeError, "positions are int32", pos=pos.half())
    bad(TypeError, "inv_freq is float64", f=f.float())
    bad(ValueError, "inv_freq is", f=f[:7])
    bad(ValueError, "pairs of a head", sections=(4, 5), f=sage.rotary_frequencies((4, 5)))
    bad(ValueError, "sections", sections=(-1, 9))
    bad(ValueError, "1 to 8 axes", sections=())
    bad(ValueError, "pairs of a head", sections=(0, 0))
    bad(RuntimeError, "no gradient", pos=pos.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="bases"):
        sage.rotary_frequencies((3, 5), base=(1e4,))


def test_decay_attention_refusals():
    q, k, v = _qkv()

    def bad(err, match, q=q, k=k, v=v, ld=LD, **kw):
        with pytest.raises(err, match=match):
            sage.decay_attention(q, k, v, ld, **kw)
    bad(TypeError, "float32 or bfloat16", q=q.half(), k=k.half(), v=v.half())
    bad(TypeError, "q, k and v are", v=v.bfloat16())
    bad(ValueError, "batch, tokens", q=q[0], k=k[0], v=v[0])
    bad(ValueError, "do not fit", k=k[:, :4])
    bad(ValueError, "do not fit", k=k[..., :8])
    bad(ValueError, "do not fit", v=v[:, :, :1])
    bad(ValueError, "4 heads over 3 key heads", k=torch.zeros(2, 5, 3, 16), v=torch.zeros(2, 5, 3, 8))
    bad(ValueError, "head sizes are 1 to 128", q=torch.zeros(2, 5, 4, 130), k=torch.zeros(2, 5, 2, 130))
    bad(ValueError, "head sizes are 1 to 128", v=torch.zeros(2, 5, 2, 0))
    bad(ValueError, r"log_decay is \[4\]", ld=torch.zeros(2))
    bad(TypeError, "log_decay is float32", ld=LD.double())
    bad(RuntimeError, "no gradient", ld=torch.zeros(4, requires_grad=True))
    bad(TypeError, "state is float32", state=torch.zeros(2, 4, 16, 8).bfloat16())
    bad(ValueError, "the state is", state=torch.zeros(2, 2, 16, 8))
    bad(TypeError, "lengths are int32", lengths=torch.zeros(2))
    bad(ValueError, "lengths are", lengths=torch.zeros(3, dtype=torch.int32))


def test_step_refusals():
    q, k, v = (t[:, 0] for t in _qkv())
    state = torch.zeros(2, 4, 16, 8)

    def bad(err, match, q=q, k=k, v=v, state=state):
        with pytest.raises(err, match=match):
            sage.decay_attention_step(q, k, v, LD, state)
    bad(ValueError, "batch, heads", q=q[None], k=k[None], v=v[None])
    bad(ValueError, "the state is", state=state[:1])
    bad(TypeError, "state is float32", state=state.bfloat16())
    bad(ValueError, "contiguous", state=torch.zeros(2, 4, 8, 16).transpose(2, 3))
    bad(RuntimeError, "no gradient", q=q.clone().requires_grad_(True))
    bad(RuntimeError, "no gradient", state=state.clone().requires_grad_(True))


def test_encoder_refusals():
    with pytest.raises(ValueError, match="heads"):
        sage.DecayEncoder(6, 96, num_heads=5)
    with pytest.raises(ValueError, match="even"):
        sage.DecayEncoder(6, 9, num_heads=3)
    with pytest.raises(ValueError, match="expected"):
        sage.DecayEncoder(6, 96)(torch.zeros(2, 3, 7))
    for sections in ((), (0, 0), (4, 5), (-1, 3)):
        with pytest.raises(ValueError, match="sections"):
            sage.DecayEncoder(6, 96, sections=sections)


def test_encoder_tables_do_not_follow_the_default_device():
    """A module built on "meta" (its parameters are filled later) still has its decays and frequencies, and a
    pickled one leaves what it keeps for a device behind."""
    import pickle
    with torch.device("meta"):
        enc = sage.DecayEncoder(6, 96, sections=(2, 3, 3))
    like = sage.DecayEncoder(6, 96, sections=(2, 3, 3))
    assert enc.qkv.weight.is_meta and enc.init_state(3)[0].is_meta
    for a, b in zip(enc._tables(torch.device("cpu")), like._tables(torch.device("cpu"))):
        assert torch.equal(a, b)
    assert like._on and not pickle.loads(pickle.dumps(like))._on and like._on


def test_encoder_tables_made_under_inference_mode_can_be_saved():
    enc = sage.DecayEncoder(6, 96)
    move = torch.Tensor.to
    with torch.inference_mode(), pytest.MonkeyPatch.context() as patch:
        patch.setattr(torch.Tensor, "to", lambda t, device: move(t, device, copy=True))
        tables = enc._tables(torch.device("cpu"))
    assert not any(t.is_inference() for t in tables)


def test_c_entries_refuse_before_any_launch():
    """Null pointers and bad shapes come back as a status with a message."""
    from sldm_sage import _lib
    lib = _lib.load()
    assert lib.sldm_layer_norm_fwd(0, None, 8, 4, 8, None, None, 1e-5, None, None, None, None) == 1
    assert b"null argument" in lib.sldm_last_error()
    assert lib.sldm_layer_norm_fwd(7, None, 8, 4, 8, None, None, 1e-5, None, None, None, None) == 1
    assert lib.sldm_layer_norm_fwd(0, None, 8, 4, 0, None, None, 1e-5, None, None, None, None) == 1
    assert lib.sldm_layer_norm_bwd(0, None, 8, None, 8, 4, 8, None, None, None, None, None, None, None, 0, None) == 0
    assert lib.sldm_layer_norm_bwd_workspace_bytes(0, 4, 8) > 0
    assert lib.sldm_decay_attention_states_bytes(0, 1, 10, 2, 2, 200, 16) == 0
    assert b"head sizes" in lib.sldm_last_error()
    assert lib.sldm_decay_attention_fwd(0, None, None, None, None, None, None, 1, 4, 2, 2, 16, 16, None, 1.0, None,
                                        None, 0, None, None, None, 0, None) == 1
    assert lib.sldm_decay_attention_step(1, None, None, None, None, None, None, 1, 3, 2, 16, 16, None, 1.0, None,
                                         None, None) == 1
    assert b"3 heads over 2" in lib.sldm_last_error()
    assert lib.sldm_decay_attention_states_bytes(1, 1 << 22, 100, 1, 1, 8, 8) == 0
    assert b"too many" in lib.sldm_last_error()
    assert lib.sldm_decay_attention_fwd(0, None, None, None, None, None, None, 1 << 20, 1, 8, 8, 8, 8, None, 1.0,
                                        None, None, 0, None, None, None, 0, None) == 1
    # long axes need room for their segments' states
    assert lib.sldm_decay_attention_states_bytes(1, 1, 100000, 1, 1, 64, 64) > 64 * 64 * 4 * 8
    assert lib.sldm_decay_attention_bwd_workspace_bytes(1, 1, 100000, 1, 1, 64, 64) > 64 * 64 * 4 * 8
    assert lib.sldm_decay_attention_states_bytes(1, 4096, 100, 6, 6, 16, 16) == 0
