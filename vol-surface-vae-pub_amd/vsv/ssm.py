"""Selective state space memory: the short causal convolution, the scan behind it, and both for single tokens.

A memory for sequences beside the LSTM / GRU / RNN ones, whose work over time is parallel:

    delta_t = softplus(dt_t + dt_bias)                               a time step per channel, from the input
    h_t     = exp(delta_t a) h_{t-1} + delta_t x_t b_t               N states per channel
    y_t     = (c_t . h_t + skip x_t) silu(gate_t)

short_conv / ssm_scan take whole sequences (and have gradients), short_conv_step / ssm_step one new token of every sequence
and update the states in place; a prompt's returned states continue in either.  SsmMemory is the module they make up,
called as nn.LSTM(batch_first=True) is.

Sequences are (B, T, D) GPU tensors in float32, bfloat16 or float16 (one type per call); b and c are (B, T, N) or, for G
groups of channels, (B, T, G, N).  Views are read in place while their last dimension is contiguous, and copied otherwise.
Weights and states are float32.  `lengths` (B) makes rows [lengths[b], T) padding: never read (whatever they hold), outputs
and gradients zero there, states taken at the length; a length outside [0, T] counts as the nearest of the two.
"""
from __future__ import annotations

import math

import torch

from . import lib as _lib
from . import native as _native


def _not_a_tensor(name, error, named):
    """What the native side's signature could not take, named if it is not a tensor where one is wanted."""
    for k, t in named.items():
        if not isinstance(t, torch.Tensor) and not (t is None and k not in ("x", "weight", "dt", "a", "b", "c", "state")):
            return ValueError(f"{name}: {k} must be a tensor, not {t!r}")
    return error


def short_conv(x, weight, bias=None, *, silu=True, initial_state=None, lengths=None, return_state=False):
    """y[:, t] = act(bias + sum_k weight[:, k] x[:, t - K + 1 + k]) per channel, act = silu or (silu=False) nothing.

    x (B, T, D), weight (D, K) with 1 to 4 taps, bias (D).  initial_state (B, K - 1, D): the inputs before the first (zeros
    without it).  Returns y (B, T, D) [, the last K - 1 inputs (B, K - 1, D) in float32]."""
    try:
        out = _native.load().short_conv(x, weight, bias, silu, initial_state, lengths, return_state)
    except TypeError as e:
        raise _not_a_tensor("short_conv", e, dict(x=x, weight=weight, bias=bias, initial_state=initial_state, lengths=lengths)) from None
    return (out[0], out[1]) if return_state else out[0]


def short_conv_step(x, state, weight, bias=None, *, silu=True):
    """short_conv for one new token of every row: x (B, D) -> y (B, D); state (B, K - 1, D), contiguous float32, is updated in
    place.  No gradients.  Bit for bit what short_conv gives for the same inputs."""
    try:
        return _native.load().short_conv_step(x, state, weight, bias, silu)
    except TypeError as e:
        raise _not_a_tensor("short_conv_step", e, dict(x=x, state=state, weight=weight, bias=bias)) from None


def ssm_scan(x, dt, a, b, c, skip=None, gate=None, *, dt_bias=None, softplus=True, initial_state=None, lengths=None,
             return_state=False):
    """The selective scan over whole sequences: x, dt [, gate] (B, T, D), a (D, N) with 1 to 16 states (negative where the
    state is to decay), b, c (B, T, [G,] N), skip, dt_bias (D).  softplus=False takes dt + dt_bias as the time step itself.
    initial_state (B, D, N).  Returns y (B, T, D) [, the state behind the last step (B, D, N) in float32].

    For gradients the states before every eighth step are kept (in float32: N / 2 bytes per element of x, N rounded up to
    4, 8 or 16).  A training step captured into a HIP graph wants parameters without a live eager graph of their own, as any
    captured backward pass of torch's does."""
    try:
        out = _native.load().ssm_scan(x, dt, a, b, c, skip, gate, dt_bias, softplus, initial_state, lengths, return_state)
    except TypeError as e:
        raise _not_a_tensor("ssm_scan", e, dict(x=x, dt=dt, a=a, b=b, c=c, skip=skip, gate=gate, dt_bias=dt_bias,
                                                initial_state=initial_state, lengths=lengths)) from None
    return (out[0], out[1]) if return_state else out[0]


def ssm_step(x, dt, a, b, c, skip=None, gate=None, *, state, dt_bias=None, softplus=True):
    """ssm_scan for one new token of every row: x, dt [, gate] (B, D), b, c (B, [G,] N) -> y (B, D); state (B, D, N),
    contiguous float32, is updated in place.  No gradients."""
    try:
        return _native.load().ssm_step(x, dt, a, b, c, skip, gate, state, dt_bias, softplus)
    except TypeError as e:
        raise _not_a_tensor("ssm_step", e, dict(x=x, dt=dt, a=a, b=b, c=c, skip=skip, gate=gate, state=state, dt_bias=dt_bias)) from None


def _padding_cleared(x, lengths):
    """Zeros behind every row's length: a projection reads those rows, and its weights' gradient would be 0 times what they hold."""
    if not isinstance(lengths, torch.Tensor) or lengths.shape != x.shape[:1] or lengths.device != x.device:
        return x                                                           # (none, or short_conv's to refuse)
    padding = torch.arange(x.shape[1], device=x.device) >= lengths[:, None]
    return x.masked_fill(padding.unsqueeze(-1), 0.0)


# ---- the memory they make up -------------------------------------------------------------------------------------

class SsmMemory(torch.nn.Module):
    """A sequence memory called as nn.LSTM(batch_first=True) is: forward(x (B, T, input_size), state=None, lengths=None) ->
    (y (B, T, hidden_size), state), state = (the convolution's (B, taps - 1, hidden_size), the scan's
    (B, hidden_size, state_size)); rows behind a length may hold anything.  step(x (B, input_size), state) takes one new token and updates the state in place."""

    def __init__(self, input_size, hidden_size, state_size=16, taps=4, dt_rank=None):
        super().__init__()
        if not 1 <= state_size <= _lib.VSV_SSM_MAX_STATE or not 1 <= taps <= _lib.VSV_CONV_MAX_TAPS:
            raise ValueError(f"SsmMemory: 1 to {_lib.VSV_SSM_MAX_STATE} states and 1 to {_lib.VSV_CONV_MAX_TAPS} taps are built")
        self.hidden_size, self.state_size, self.taps = hidden_size, state_size, taps
        self.dt_rank = dt_rank or max(1, -(-hidden_size // 16))
        self.in_proj = torch.nn.Linear(input_size, 2 * hidden_size)
        self.x_proj = torch.nn.Linear(hidden_size, self.dt_rank + 2 * state_size, bias=False)
        self.dt_proj = torch.nn.Linear(self.dt_rank, hidden_size, bias=False)
        bound = 1.0 / math.sqrt(taps)
        self.conv_weight = torch.nn.Parameter(torch.empty(hidden_size, taps).uniform_(-bound, bound))
        self.conv_bias = torch.nn.Parameter(torch.zeros(hidden_size))
        step = torch.exp(torch.empty(hidden_size).uniform_(math.log(1e-3), math.log(1e-1)))
        self.dt_bias = torch.nn.Parameter(torch.log(torch.expm1(step)))    # time steps of 0.001 to 0.1 at the start
        self.a_log = torch.nn.Parameter(torch.log(torch.arange(1.0, state_size + 1.0)).repeat(hidden_size, 1))
        self.skip = torch.nn.Parameter(torch.ones(hidden_size))

    def _projected(self, x):
        r, n = self.dt_rank, self.state_size
        dt, b, c = self.x_proj(x).split([r, n, n], dim=-1)
        return self.dt_proj(dt), b, c

    def forward(self, x, state=None, lengths=None):
        x, gate = self.in_proj(_padding_cleared(x, lengths)).chunk(2, dim=-1)
        conv, scan = state if state is not None else (None, None)
        x, conv = short_conv(x, self.conv_weight.float(), self.conv_bias.float(), initial_state=conv, lengths=lengths, return_state=True)
        dt, b, c = self._projected(x)
        y, scan = ssm_scan(x, dt, -torch.exp(self.a_log.float()), b, c, self.skip.float(), gate, dt_bias=self.dt_bias.float(),
                           initial_state=scan, lengths=lengths, return_state=True)
        return y, (conv, scan)

    @torch.no_grad()
    def step(self, x, state):
        x, gate = self.in_proj(x).chunk(2, dim=-1)
        x = short_conv_step(x, state[0], self.conv_weight.float(), self.conv_bias.float())
        dt, b, c = self._projected(x)
        return ssm_step(x, dt, -torch.exp(self.a_log.float()), b, c, self.skip.float(), gate, state=state[1], dt_bias=self.dt_bias.float())
