"""Layers beside ParaConv2d: dropout, a short causal convolution, a state
space scan, linear attention and group norm, each as a function and as a module.

They take [batch, channels, length] tensors: the map [N, C, H, W] of a
convolution layer is one with ``x.flatten(2)``, and goes back with
``view(N, C, H, W)``, without a copy.

* :func:`dropout` / :class:`Dropout`: elements kept or dropped by a
  counter-based generator; the mask is computed again in the backward pass and
  never stored.  Optionally added to a residual in the same pass.
* :func:`causal_conv` / :class:`CausalConv`: one filter of up to 8 taps per
  channel over a token and those before it; :func:`causal_conv_step` for one
  token of each request.
* :func:`ssm_scan` / :class:`SSMScan`: a diagonal linear recurrence whose decay
  and inputs depend on the token; :func:`ssm_scan_step` for one token of each
  request.
* :func:`linear_attention` / :class:`LinearAttention`: a matrix state for each
  head, with a decay; :func:`linear_attention_step` for one token of each
  request.
* :func:`group_norm` / :class:`GroupNorm`: over groups of channels, with an
  optional SiLU, in both orders of dimensions.

CUDA tensors only (float32, float16 and bfloat16; dropout float64 too), on the
current stream of the tensors' device; sums and states in 32 bits.  Results
and gradients are deterministic.  Dropout is differentiable any number of
times, the others once; forward-mode derivatives are refused.  All of it,
backward passes too, can be captured into CUDA graphs; as for every backward
pass, leaves that still belong to an eager autograd graph made on another
stream must be released (or their graph run on the capturing stream) before
that.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from ._lib import load_op_library

load_op_library()


class _ops:
    """The C++ ops, their overloads looked up once."""

    dropout = torch.ops.paraconv2d_b200.dropout.default
    dropout_next_key = torch.ops.paraconv2d_b200.dropout_next_key.default
    causal_conv_forward = torch.ops.paraconv2d_b200.causal_conv_forward.default
    causal_conv_step = torch.ops.paraconv2d_b200.causal_conv_step.default
    ssm_scan_forward = torch.ops.paraconv2d_b200.ssm_scan_forward.default
    ssm_scan_step = torch.ops.paraconv2d_b200.ssm_scan_step.default
    linear_attention_forward = torch.ops.paraconv2d_b200.linear_attention_forward.default
    linear_attention_step = torch.ops.paraconv2d_b200.linear_attention_step.default
    group_norm_forward = torch.ops.paraconv2d_b200.group_norm_forward.default


def _silu(activation) -> bool:
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return activation == "silu"


# -------------------------------------------------------------------- dropout

def dropout(x: Tensor, p: float, key: Tensor, residual: Optional[Tensor] = None) -> Tensor:
    """``x`` with each element dropped with probability ``p`` and the others
    divided by the probability of being kept, plus ``residual``.

    ``key``: int64 [2] on the GPU, the seed and an offset.  The same key drops
    the same elements (by their place in the contiguous order of ``x``), on any
    device and for any type; calls that should differ need keys that differ in
    either number (:class:`Dropout` makes them).  ``p`` is rounded to a
    multiple of 2^-16, and the scale is the inverse of the rounded
    probability.  A dropped element is 0, whatever it held.
    """
    return _ops.dropout(x, key, p, residual)


class Dropout(nn.Module):
    """:func:`dropout` in training, the identity (plus the residual) in
    evaluation.  Every call in training uses the next offset of ``seed``, kept
    on the GPU in the buffer ``state`` and counted there (by a small launch of
    its own): a call that a CUDA graph replays drops other elements each time, and a checkpoint goes on
    where it was saved.  Ranks of a data-parallel job need seeds of their own,
    and so have layers whose masks should not be the same; a wrapper that
    broadcasts buffers would give all ranks the same seed.  Where activations
    are computed again in the backward pass, a second call would drop other
    elements: take a key before, and call :func:`dropout` with it."""

    def __init__(self, p: float = 0.5, seed: int = 0, device=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1], got {p}")
        self.p = float(p)
        self.register_buffer("state", torch.tensor([seed, 0], dtype=torch.int64, device=device))

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        return dropout(x, self.p, _ops.dropout_next_key(self.state), residual)

    def extra_repr(self) -> str:
        return f"p={self.p}"


# --------------------------------------------------------- causal convolution

def causal_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
                initial_state: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                return_final_state: bool = False):
    """Convolution of each channel of ``x`` [batch, channels, length] with its
    filter ``weight`` [channels, taps] over a token and the ``taps - 1`` before
    it (``weight[:, -1]`` meets the token itself), plus ``bias`` [channels],
    through ``activation`` (None or 'silu').

    ``initial_state`` [batch, channels, taps-1]: the inputs before the first
    token (zeros if None).  ``lengths`` (int32 [batch], on the GPU): the tokens
    of each row; what lies behind them is not read, and outputs and gradients
    there are 0.  Returns the output, and with ``return_final_state`` the pair
    (output, the last taps-1 inputs of each row).  1 to 8 taps; weight and bias
    of x's type or float32.
    """
    outs = _ops.causal_conv_forward(x, weight, bias, initial_state, lengths, _silu(activation),
                                    bool(return_final_state))
    return (outs[0], outs[1]) if return_final_state else outs[0]


def causal_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor] = None,
                     activation: Optional[str] = None, slots: Optional[Tensor] = None) -> Tensor:
    """:func:`causal_conv` of one token for each row of ``x`` [batch,
    channels], with the inputs before it in ``state`` [places, channels,
    taps-1], which is moved on in place.  Row b uses place ``slots[b]`` (int32
    [batch], on the GPU), or place b without slots.  A slot of -1 marks a row
    without a request: its output is 0 and no state changes.  A slot outside
    the states, or one that an earlier row has too, makes the row NaN and
    changes no state.  Inputs that share memory with ``state`` are refused."""
    return _ops.causal_conv_step(x, state, weight, bias, slots, _silu(activation))


class CausalConv(nn.Module):
    """:func:`causal_conv` with its ``weight`` [channels, taps] and ``bias``."""

    def __init__(self, channels: int, taps: int = 4, bias: bool = True, activation: Optional[str] = None, device=None,
                 dtype=None):
        super().__init__()
        if not 1 <= taps <= 8:
            raise ValueError(f"taps must be 1 to 8, got {taps}")
        _silu(activation)
        kw = dict(device=device, dtype=dtype)
        self.channels, self.taps, self.activation = channels, taps, activation
        bound = 1 / math.sqrt(taps)
        self.weight = nn.Parameter(torch.empty(channels, taps, **kw).uniform_(-bound, bound))
        self.bias = nn.Parameter(torch.empty(channels, **kw).uniform_(-bound, bound)) if bias else None

    def new_state(self, places: int, dtype=None) -> Tensor:
        """Zero states for ``places`` requests."""
        return torch.zeros(places, self.channels, self.taps - 1, device=self.weight.device,
                           dtype=dtype or self.weight.dtype)

    def forward(self, x, initial_state=None, lengths=None, return_final_state=False):
        return causal_conv(x, self.weight, self.bias, self.activation, initial_state, lengths, return_final_state)

    @torch.no_grad()
    def step(self, x, state, slots=None):
        return causal_conv_step(x, state, self.weight, self.bias, self.activation, slots)

    def extra_repr(self) -> str:
        return f"channels={self.channels}, taps={self.taps}, activation={self.activation}"


# ----------------------------------------------------------- state space scan

def ssm_scan(u: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor] = None,
             z: Optional[Tensor] = None, delta_bias: Optional[Tensor] = None, delta_softplus: bool = False,
             initial_state: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
             return_final_state: bool = False):
    """The recurrence, for each channel and each of its states n::

        d_t = delta_t + delta_bias            (softplus of it with delta_softplus)
        h_t[n] = exp(d_t A[n]) h_{t-1}[n] + d_t u_t B_t[n]
        out_t = (sum_n C_t[n] h_t[n] + D u_t) * silu(z_t)

    ``u``, ``delta`` and ``z`` (None: no gate): [batch, channels, length];
    ``B`` and ``C``: [batch, groups, states, length], each group for
    channels/groups neighbouring channels; all of one type.  ``A`` [channels,
    states], ``D`` and ``delta_bias`` [channels] (None: 0) and the states
    [batch, channels, states] are float32.  1 to 128 states; up to 2^24 rows
    (batch times channels) and 2^30 tokens.  A of -inf forgets at every token.

    ``initial_state`` (None: 0), ``lengths`` and ``return_final_state`` as for
    :func:`causal_conv`.  Gradients reach every tensor but ``lengths``.  For
    the backward pass the forward one keeps the states of every 16th or 32nd
    token in float32: 2 bytes per channel and token with 16 states, 32 with
    128.  The backward pass itself takes scratch of about states^2 / 64 bytes
    per channel and token: 4 with 16 states, but 64 with 64 and 256 with 128.
    """
    outs = _ops.ssm_scan_forward(u, delta, A, B, C, D, z, delta_bias, initial_state, lengths, bool(delta_softplus),
                                 bool(return_final_state), False)
    return (outs[0], outs[1]) if return_final_state else outs[0]


def ssm_scan_step(u: Tensor, delta: Tensor, state: Tensor, A: Tensor, B: Tensor, C: Tensor,
                  D: Optional[Tensor] = None, z: Optional[Tensor] = None, delta_bias: Optional[Tensor] = None,
                  delta_softplus: bool = False, slots: Optional[Tensor] = None) -> Tensor:
    """:func:`ssm_scan` of one token for each row: ``u``, ``delta``, ``z``
    [batch, channels], ``B``, ``C`` [batch, groups, states]; ``state`` float32
    [places, channels, states] is moved on in place, with ``slots`` as for
    :func:`causal_conv_step`."""
    return _ops.ssm_scan_step(u, delta, state, A, B, C, D, z, delta_bias, slots, bool(delta_softplus))


class SSMScan(nn.Module):
    """:func:`ssm_scan` with softplus and its parameters: ``A_log`` [channels,
    states] (A = -exp(A_log), decays of 1 to ``states`` at first), ``D`` and
    ``delta_bias`` [channels] (steps from 0.001 to 0.1 at first).  delta, B and
    C come with each call: projections of the input make them.  Every call
    makes A from A_log, by two small launches before its own; a loop over
    tokens may make A once and call :func:`ssm_scan_step` with it."""

    def __init__(self, channels: int, states: int = 16, device=None):
        super().__init__()
        if not 1 <= states <= 128:
            raise ValueError(f"states must be 1 to 128, got {states}")
        self.channels, self.states = channels, states
        decay = torch.arange(1, states + 1, device=device, dtype=torch.float32)
        self.A_log = nn.Parameter(torch.log(decay).repeat(channels, 1))
        self.D = nn.Parameter(torch.ones(channels, device=device))
        step = torch.exp(torch.rand(channels, device=device) * math.log(100.0) + math.log(0.001))
        self.delta_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))  # softplus gives `step`

    def new_state(self, places: int) -> Tensor:
        """Zero states for ``places`` requests."""
        return torch.zeros(places, self.channels, self.states, device=self.A_log.device)

    def _params(self):
        # float32 also in a module that was moved to a 16-bit type
        return -torch.exp(self.A_log.float()), self.D.float(), self.delta_bias.float()

    def forward(self, u, delta, B, C, z=None, initial_state=None, lengths=None, return_final_state=False):
        A, D, delta_bias = self._params()
        return ssm_scan(u, delta, A, B, C, D, z, delta_bias, True, initial_state, lengths, return_final_state)

    @torch.no_grad()
    def step(self, u, delta, state, B, C, z=None, slots=None):
        A, D, delta_bias = self._params()
        return ssm_scan_step(u, delta, state, A, B, C, D, z, delta_bias, True, slots)

    def extra_repr(self) -> str:
        return f"channels={self.channels}, states={self.states}"


# ----------------------------------------------------------- linear attention

def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, scale: Optional[float] = None,
                     initial_state: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
                     return_final_state: bool = False):
    """The recurrence, for each head::

        S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T        (keys x values)
        out_t = scale S_t^T q_t

    ``q`` and ``k``: [batch, groups, keys, length], each group for
    heads/groups neighbouring heads; ``v`` and the result: [batch, heads,
    values, length]; of one type.  ``log_decay``: float32, [heads] or [batch,
    heads, length], at most 0 in use (-inf forgets all before a token).
    ``scale``: keys^-0.5 if None.  States [batch, heads, keys, values] are
    float32.  1 to 128 keys and values; up to 2^20 heads of rows and 2^30
    tokens.

    ``initial_state`` (None: 0), ``lengths`` and ``return_final_state`` as for
    :func:`causal_conv`.  Gradients reach every tensor but ``lengths``.  For
    the backward pass the forward one keeps the states of every 64th token
    (every 32nd in float32 and float16), keys*values/16 bytes (/8) per head and
    token, and the backward pass takes as much again.
    """
    scale = q.shape[-2] ** -0.5 if scale is None else float(scale)
    outs = _ops.linear_attention_forward(q, k, v, log_decay, initial_state, lengths, scale, bool(return_final_state),
                                         False)
    return (outs[0], outs[1]) if return_final_state else outs[0]


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor,
                          scale: Optional[float] = None, slots: Optional[Tensor] = None) -> Tensor:
    """:func:`linear_attention` of one token for each row: ``q``, ``k`` [batch,
    groups, keys], ``v`` [batch, heads, values], ``log_decay`` [heads] or
    [batch, heads]; ``state`` float32 [places, heads, keys, values] is moved on
    in place, with ``slots`` as for :func:`causal_conv_step`."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    return _ops.linear_attention_step(q, k, v, log_decay, state, slots, scale)


class LinearAttention(nn.Module):
    """:func:`linear_attention` with a decay for each head as its parameter
    ``rate`` [heads] (log_decay = -exp(rate)): memories of 32 to 4096 tokens
    over the heads at first.  q, k and v come with each call: projections of
    the input make them.  Where decays come with the tokens too, call the
    function."""

    def __init__(self, heads: int, keys: int, values: int, scale: Optional[float] = None, device=None):
        super().__init__()
        if heads < 1 or not 1 <= keys <= 128 or not 1 <= values <= 128:
            raise ValueError(f"heads must be positive, keys and values 1 to 128, got {heads}, {keys} and {values}")
        self.heads, self.keys, self.values, self.scale = heads, keys, values, scale
        spread = torch.linspace(5, 12, heads, device=device, dtype=torch.float32)
        self.rate = nn.Parameter(torch.log(-torch.log1p(-torch.exp2(-spread))))

    def new_state(self, places: int) -> Tensor:
        """Zero states for ``places`` requests."""
        return torch.zeros(places, self.heads, self.keys, self.values, device=self.rate.device)

    def _log_decay(self):
        return -torch.exp(self.rate.float())  # float32 also in a module that was moved to a 16-bit type

    def forward(self, q, k, v, initial_state=None, lengths=None, return_final_state=False):
        return linear_attention(q, k, v, self._log_decay(), self.scale, initial_state, lengths, return_final_state)

    @torch.no_grad()
    def step(self, q, k, v, state, slots=None):
        return linear_attention_step(q, k, v, self._log_decay(), state, self.scale, slots)

    def extra_repr(self) -> str:
        return f"heads={self.heads}, keys={self.keys}, values={self.values}"


# ----------------------------------------------------------------- group norm

def group_norm(x: Tensor, groups: int, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None,
               eps: float = 1e-5, activation: Optional[str] = None, lengths: Optional[Tensor] = None) -> Tensor:
    """``x`` [batch, channels, ...] less its mean and divided by its deviation
    over each of ``groups`` equal groups of neighbouring channels and all
    positions of a batch row, times ``weight`` plus ``bias`` [channels] (None:
    1 and 0; x's type or float32), through ``activation`` (None or 'silu').

    ``x`` is taken as it lies, contiguous or channels last (the memory format,
    or any [batch, channels, length] view of [batch, length, channels]), and
    the result lies likewise; in another order it is copied.  ``lengths``
    (int32 [batch], on the GPU; for [batch, channels, length] only): the
    tokens of each row; what lies behind them is not read and counts nothing,
    and outputs and gradients there are 0.  Up to 8192 channels a group.
    """
    return _ops.group_norm_forward(x, weight, bias, lengths, groups, eps, _silu(activation), False)[0]


class GroupNorm(nn.Module):
    """:func:`group_norm` with its ``weight`` and ``bias`` [channels]."""

    def __init__(self, groups: int, channels: int, eps: float = 1e-5, affine: bool = True,
                 activation: Optional[str] = None, device=None, dtype=None):
        super().__init__()
        if groups < 1 or channels % groups:
            raise ValueError(f"channels ({channels}) must be a multiple of groups ({groups})")
        _silu(activation)
        self.groups, self.channels, self.eps, self.activation = groups, channels, eps, activation
        kw = dict(device=device, dtype=dtype)
        self.weight = nn.Parameter(torch.ones(channels, **kw)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels, **kw)) if affine else None

    def forward(self, x, lengths=None):
        return group_norm(x, self.groups, self.weight, self.bias, self.eps, self.activation, lengths)

    def extra_repr(self) -> str:
        return f"groups={self.groups}, channels={self.channels}, eps={self.eps}, activation={self.activation}"
