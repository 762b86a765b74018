"""Operators of a trajectory encoder without a GRU, on gfx950 kernels.

GruSage reads each vehicle's frames with a GRU (grusage.py:66-71, :160-161;
:class:`sldm_sage.GRU` here), one frame after the other.  These operators mix
the frames of a sequence at once and keep the GRU's contract, a state that goes
in and comes out, so live data can go on frame by frame:

    layer_norm(x, weight, bias, eps)                layer norm, its gradients
    rotary_axes(q, k, positions, inv_freq, sections)  time, x and y as angles
    decay_attention(q, k, v, log_decay, ...)        linear attention whose state
                                                    fades by a factor a head
    decay_attention_step(q, k, v, log_decay, state) one token of it, in place

:class:`LayerNorm` and :class:`DecayEncoder` are the modules over them.  All
run on ROCm tensors in float32 or bfloat16 on the current stream; CPU tensors
raise (no fallback), and so do second and forward-mode derivatives.  Kernels: csrc/norm.hip, rotary.hip, decay.hip; operators
with their autograd: csrc/sequence_ops.cpp (``torch.ops.sldm``).
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import torch_ops

_ops = None


def _sldm():
    global _ops
    if _ops is None:
        o = torch_ops.load()
        _ops = (o.layer_norm.default, o.rotary_axes.default, o.decay_attention.default,
                o.decay_attention_step.default)
    return _ops


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    ``x``: any shape, float32 or bfloat16; ``weight`` / ``bias``: ``[x.size(-1)]``, float32 or
    x's dtype.  Statistics and the columns' gradient sums are float32, in a fixed order."""
    return _sldm()[0](x, weight, bias, eps)


def rotary_frequencies(sections, base=10000.0, device=None) -> torch.Tensor:
    """float64 ``[sum(sections)]``: a frequency ladder ``base ** (-j / n)``, ``j = 0 .. n - 1``,
    for each axis of ``n`` pairs.  ``base``: a number, or one for each axis."""
    sections = [int(n) for n in sections]
    bases = [float(base)] * len(sections) if isinstance(base, (int, float)) else [float(b) for b in base]
    if len(bases) != len(sections):
        raise ValueError(f"rotary_frequencies: {len(bases)} bases for {len(sections)} axes")
    f = [b ** (-j / n) for n, b in zip(sections, bases) for j in range(n)]
    return torch.tensor(f, dtype=torch.float64, device=device)


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                inv_freq: torch.Tensor, sections, interleaved: bool = False):
    """Turn the pairs of each head of ``q`` and ``k`` by ``positions * inv_freq``.

    ``q`` ``[.., tokens, heads, D]``, ``k`` the same with its own heads (or None), ``positions``
    ``[.., tokens, axes]`` (int32, int64, float32 or float64: frames, metres, rows and columns),
    ``inv_freq`` float64 ``[P]``, ``P = sum(sections) <= D / 2``.  Axis 0 turns the first
    ``sections[0]`` pairs, axis 1 the next ``sections[1]``, and so on; pair p is columns
    ``(p, p + P)``, or ``(2p, 2p + 1)`` if ``interleaved``; columns from ``2P`` on stay.  Angles are
    computed in float64.  Returns new ``(q, k)``; differentiable in q and k."""
    oq, ok = _sldm()[1](q, k, positions, inv_freq, sections, interleaved)
    return oq, ok if k is not None else None


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                    scale: float | None = None, state: torch.Tensor | None = None,
                    lengths: torch.Tensor | None = None):
    """Linear attention with a decay for each head; returns ``(out, state)``.

        S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T        out_t = scale q_t S_t

    ``q`` ``[B, T, H, Dk]``, ``k`` ``[B, T, Hk, Dk]``, ``v`` ``[B, T, Hk, Dv]`` (float32 or
    bfloat16; ``Hk`` divides ``H``, head h reads key head ``h // (H // Hk)``; sizes 1 to 128;
    ``B * H`` below 2^22);
    ``log_decay`` float32 ``[H]``, not above 0; ``scale`` defaults to ``Dk ** -0.5``; ``state``
    float32 ``[B, H, Dk, Dv]`` is the state before the first token (None: zeros) and the returned
    one that behind the last.  ``lengths`` (int32 or int64 ``[B]``, clamped to ``[0, T]``): later
    tokens are padding, whatever they hold: outputs and gradients there are zeros and the state
    ends before them.  An infinity or NaN reaches what these sums say and no token before its own.
    Differentiable in q, k, v and state."""
    return _sldm()[2](q, k, v, log_decay, state, lengths, scale)


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         log_decay: torch.Tensor, state: torch.Tensor,
                         scale: float | None = None) -> torch.Tensor:
    """One token of :func:`decay_attention` for each sequence, for live data.

    ``q`` ``[B, H, Dk]``, ``k`` ``[B, Hk, Dk]``, ``v`` ``[B, Hk, Dv]``; ``state`` float32
    ``[B, H, Dk, Dv]``, contiguous, is moved on in place.  Returns ``out [B, H, Dv]``; has no
    gradient."""
    return _sldm()[3](q, k, v, log_decay, state, scale)


class LayerNorm(nn.Module):
    """``torch.nn.LayerNorm`` over the last dimension (same parameters and names) on gfx950 kernels."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None):
        super().__init__()
        shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
        if len(shape) != 1:
            raise ValueError(f"sldm_sage.LayerNorm normalises the last dimension only, got {shape}")
        self.normalized_shape, self.eps, self.elementwise_affine = shape, eps, elementwise_affine
        fk = dict(device=device, dtype=dtype)
        self.weight = nn.Parameter(torch.ones(shape, **fk)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(shape, **fk)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() == 0 or x.size(-1) != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm: expected [.., {self.normalized_shape[0]}], got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.normalized_shape}, eps={self.eps}, elementwise_affine={self.elementwise_affine}"


class DecayEncoder(nn.Module):
    """A trajectory encoder in the GRU's place: norm, projection, rotary positions, decay attention, norm.

    ``out, state = encoder(x, state=None, positions=None, lengths=None)`` with ``x``
    ``[N, T, input_size]`` and ``out`` ``[N, T, hidden_size]`` (compare ``GRU(batch_first=True)``,
    grusage.py:160-161); ``state`` ``(S [N, heads, D, D], tokens seen [N])`` goes on from an earlier
    call.  ``positions`` ``[N, T, axes]`` are the rotary positions (default: the frame's number, on
    every axis); ``sections`` says how many of the ``D / 2`` pairs each axis turns.  :meth:`step` takes
    one frame ``[N, input_size]`` and moves the state on in place.
    """

    def __init__(self, input_size: int, hidden_size: int, num_heads: int = 6, sections=None,
                 rotary_base: float = 10000.0, device=None, dtype=None):
        super().__init__()
        if num_heads < 1 or hidden_size % num_heads or not 2 <= hidden_size // num_heads <= 128 \
                or hidden_size // num_heads % 2:
            raise ValueError(f"DecayEncoder: {hidden_size} units do not make {num_heads} heads of an even "
                             "size of 2 to 128")
        self.input_size, self.hidden_size, self.num_heads = input_size, hidden_size, num_heads
        self.head_dim = hidden_size // num_heads
        self.sections = [self.head_dim // 2] if sections is None else [int(n) for n in sections]
        if not 1 <= len(self.sections) <= 8 or min(self.sections) < 0 or \
                not 1 <= sum(self.sections) <= self.head_dim // 2:
            raise ValueError(f"DecayEncoder: sections {self.sections} do not turn 1 to {self.head_dim // 2} pairs "
                             "on 1 to 8 axes")
        fk = dict(device=device, dtype=dtype)
        self.norm = LayerNorm(hidden_size, **fk)
        self.embed = nn.Linear(input_size, hidden_size, **fk)
        self.qkv = nn.Linear(hidden_size, 3 * hidden_size, bias=False, **fk)
        self.head_norm = LayerNorm(self.head_dim, elementwise_affine=False)
        self.proj = nn.Linear(hidden_size, hidden_size, bias=False, **fk)
        # fading over 4 to 4 * 2^(heads - 1) frames, and the rotary ladder: fixed, and kept in
        # their own types where the module's parameters are cast (on the host whatever the default
        # device, so that a module built on "meta" has them too)
        heads = torch.arange(num_heads, dtype=torch.float32, device="cpu")
        self._log_decay = torch.log1p(-torch.exp2(-2.0 - heads))
        self._inv_freq = rotary_frequencies(self.sections, rotary_base, device="cpu")
        self._on: dict = {}

    def _tables(self, device: torch.device):
        t = self._on.get(device)
        if t is None:
            with torch.inference_mode(False):      # kept: a later training pass saves them
                t = self._on[device] = (self._log_decay.to(device), self._inv_freq.to(device))
        return t

    def __getstate__(self):
        return {**self.__dict__, "_on": {}}        # a copy's tables follow its own device

    def _qkv(self, x, positions):
        h = F.silu(self.embed(x))
        q, k, v = self.qkv(self.norm(h)).unflatten(-1, (3, self.num_heads, self.head_dim)).unbind(-3)
        q, k = rotary_axes(q, k, positions, self._tables(x.device)[1], self.sections)
        return h, q, k, v

    def _out(self, h, o):
        return h + self.proj(self.head_norm(o).flatten(-2))

    def _state(self, state, n: int, whole: bool):
        """(S, seen) of ``n`` sequences; ``whole``: neither may be None."""
        want = [(n, self.num_heads, self.head_dim, self.head_dim), (n,)]
        ok = isinstance(state, (tuple, list)) and len(state) == 2 and all(
            t is None and not whole or isinstance(t, torch.Tensor) and tuple(t.shape) == size
            for t, size in zip(state, want))
        if not ok:
            got = tuple(tuple(t.shape) if isinstance(t, torch.Tensor) else t for t in state) \
                if isinstance(state, (tuple, list)) else type(state).__name__
            raise ValueError(f"DecayEncoder: the state is (S {list(want[0])}, tokens seen [{n}]), got {got}")
        return state

    def forward(self, x: torch.Tensor, state=None, positions: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None):
        if x.dim() != 3 or x.size(-1) != self.input_size:
            raise ValueError(f"DecayEncoder: expected [N, T, {self.input_size}], got {tuple(x.shape)}")
        N, T = x.shape[:2]
        S, seen = (None, None) if state is None else self._state(state, N, whole=False)
        if seen is None:
            seen = torch.zeros(N, dtype=torch.int64, device=x.device)
        if positions is None:
            positions = (seen[:, None] + torch.arange(T, device=x.device))[..., None].expand(
                N, T, len(self.sections))
        h, q, k, v = self._qkv(x, positions)
        o, S = decay_attention(q, k, v, self._tables(x.device)[0], state=S, lengths=lengths)
        return self._out(h, o), (S, seen + (T if lengths is None else lengths.clamp(0, T)))

    @torch.no_grad()
    def step(self, x: torch.Tensor, state, positions: torch.Tensor | None = None):
        """One frame ``x [N, input_size]``; ``state`` (of an earlier call, or :meth:`init_state`) is moved
        on in place.  Returns ``out [N, hidden_size]``."""
        if x.dim() != 2 or x.size(-1) != self.input_size:
            raise ValueError(f"DecayEncoder.step: expected [N, {self.input_size}], got {tuple(x.shape)}")
        S, seen = self._state(state, x.size(0), whole=True)
        if positions is None:
            positions = seen[:, None].expand(-1, len(self.sections))
        h, q, k, v = self._qkv(x, positions)
        o = decay_attention_step(q, k, v, self._tables(x.device)[0], S)
        seen.add_(1)
        return self._out(h, o)

    def init_state(self, n: int, device=None):
        """The state before the first frame of ``n`` sequences (``device``: the parameters')."""
        device = self.qkv.weight.device if device is None else device
        return (torch.zeros(n, self.num_heads, self.head_dim, self.head_dim, dtype=torch.float32, device=device),
                torch.zeros(n, dtype=torch.int64, device=device))
