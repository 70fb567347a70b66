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

import ctypes as C
import math

import torch

from . import lib as _lib

_GPU = "there is no CPU fallback"


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}              # VSV_F32, VSV_BF16, VSV_F16
_Tensor, _f32_type = torch.Tensor, torch.float32
_entries = {}


def _last(t):
    """t itself where its last dimension is contiguous, else a copy."""
    return t if t.is_contiguous() or t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _seq(what, name, t, shape, dtype=None):
    if not isinstance(t, _Tensor) or t.shape != shape:
        raise ValueError(f"{what}: {name} must be a tensor of shape {tuple(shape)}, not {tuple(t.shape) if isinstance(t, _Tensor) else t!r}")
    if t.dtype not in _TYPES or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{what}: {name} must be {dtype or 'float32, bfloat16 or float16'}, not {t.dtype}")
    return t if t.is_contiguous() else _last(t)


def _f32(what, name, t, shape):
    if t is None:
        return None
    if not isinstance(t, _Tensor) or t.shape != shape or t.dtype is not _f32_type:
        raise ValueError(f"{what}: {name} must be a float32 tensor of shape {tuple(shape)}"
                         + (f", not {t.dtype} {tuple(t.shape)}" if isinstance(t, _Tensor) else f", not {t!r}"))
    return t if t.is_contiguous() else t.contiguous()


def _lengths(what, t, B):
    if t is None:
        return None
    if not isinstance(t, _Tensor) or t.shape != (B,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: lengths must be an int32 or int64 tensor of shape ({B},)")
    if t.dtype == torch.int64:
        t = t.clamp(0, 2**31 - 1).to(torch.int32)
    return t.contiguous()


def _same_gpu(what, x, *others):
    if not x.is_cuda:
        raise RuntimeError(f"{what}: tensors must be on a GPU; {_GPU}")
    at = x.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            raise ValueError(f"{what}: tensors are on {t.device} and {x.device}")


def _call(name, at, *args):
    """One entry point on the current stream of GPU `at`."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    if torch._C._cuda_getDevice() == at:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(at))
    else:
        with torch.cuda.device(at):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(at))
    if rc:
        _lib.check(rc, name)


def _size(name, desc):
    """A size that the library answers for a descriptor."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(_lib.load(), name)
    return fn(desc)


def _workspace(nbytes, device):
    return torch.empty(nbytes or 16, dtype=torch.uint8, device=device)


def _wants_grad(*ts):
    if not torch.is_grad_enabled():
        return False
    for t in ts:
        if t is not None and t.requires_grad:
            return True
    return False


def _touched(t):
    """What an in-place operation leaves on a tensor that was written through its address."""
    torch.autograd.graph.increment_version(t)


# ---- short causal convolution ------------------------------------------------------------------------------------

def short_conv(x, weight, bias=None, *, silu=True, initial_state=None, lengths=None, return_state=False):
    """y[:, t] = act(bias + sum_k weight[:, k] x[:, t - K + 1 + k]) per channel, act = silu or (silu=False) nothing.

    x (B, T, D), weight (D, K) with 1 to 4 taps, bias (D).  initial_state (B, K - 1, D): the inputs before the first (zeros
    without it).  Returns y (B, T, D) [, the last K - 1 inputs (B, K - 1, D) in float32]."""
    what = "short_conv"
    if not isinstance(x, _Tensor) or x.dim() != 3:
        raise ValueError(f"{what}: x must be a tensor (B, T, D)")
    B, T, D = x.shape
    if not isinstance(weight, _Tensor) or weight.dim() != 2 or not 1 <= weight.shape[1] <= _lib.VSV_CONV_MAX_TAPS or D < 1:
        raise ValueError(f"{what}: weight must be a tensor (D, K) with 1 to {_lib.VSV_CONV_MAX_TAPS} taps")
    K = weight.shape[1]
    x = _seq(what, "x", x, (B, T, D))
    weight, bias = _f32(what, "weight", weight, (D, K)), _f32(what, "bias", bias, (D,))
    initial_state = _f32(what, "initial_state", initial_state, (B, K - 1, D))
    lengths = _lengths(what, lengths, B)
    _same_gpu(what, x, weight, bias, initial_state, lengths)
    if _wants_grad(x, weight, bias, initial_state):
        from .autograd import ShortConv
        y, state = ShortConv.apply(x, weight, bias, initial_state, lengths, bool(silu), bool(return_state))
    else:
        y, state, _ = conv_forward(x, weight, bias, initial_state, lengths, silu, return_state)
    return (y, state) if return_state else y


def conv_forward(x, weight, bias, state_in, lengths, silu, want_state):
    """The launch behind short_conv: (y, state | None, the descriptor vsv_short_conv_backward takes again)."""
    (B, T, D), K = x.shape, weight.shape[1]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    state = torch.empty((B, K - 1, D), dtype=torch.float32, device=x.device) if want_state else None
    d = _lib.VsvShortConv(_TYPES[x.dtype], K, int(silu), B, T, D, x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(),
                          _ptr(bias), _ptr(state_in), _ptr(lengths), y.data_ptr(), _ptr(state) or None)
    _call("vsv_short_conv", x.get_device(), C.byref(d))
    return y, state, d


def short_conv_step(x, state, weight, bias=None, *, silu=True):
    """short_conv for one new token of every row: x (B, D) -> y (B, D); state (B, K - 1, D), contiguous float32, is updated in
    place.  No gradients."""
    what = "short_conv_step"
    if not isinstance(x, _Tensor) or x.dim() != 2:
        raise ValueError(f"{what}: x must be a tensor (B, D)")
    B, D = x.shape
    if not isinstance(weight, _Tensor) or weight.dim() != 2 or not 1 <= weight.shape[1] <= _lib.VSV_CONV_MAX_TAPS or D < 1:
        raise ValueError(f"{what}: weight must be a tensor (D, K) with 1 to {_lib.VSV_CONV_MAX_TAPS} taps")
    K = weight.shape[1]
    x = _seq(what, "x", x, (B, D))
    weight, bias = _f32(what, "weight", weight, (D, K)), _f32(what, "bias", bias, (D,))
    _in_place(what, state, (B, K - 1, D))
    _same_gpu(what, x, weight, bias, state)
    if _wants_grad(x, weight, bias, state):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    d = _lib.VsvShortConv(_TYPES[x.dtype], K, int(silu), B, 1, D, x.data_ptr(), x.stride(0), 0, weight.data_ptr(), _ptr(bias),
                          None, None, y.data_ptr(), state.data_ptr())
    _call("vsv_short_conv_step", x.get_device(), C.byref(d))
    _touched(state)
    return y


def _in_place(what, state, shape):
    if not isinstance(state, _Tensor) or state.shape != shape or state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError(f"{what}: state must be a contiguous float32 tensor of shape {tuple(shape)} (it is updated in place)")


# ---- selective scan ----------------------------------------------------------------------------------------------

def _grouped(what, name, t, lead, D, N, dtype):
    """b or c with its group dimension."""
    if isinstance(t, _Tensor) and t.dim() == len(lead) + 1:
        t = t.unsqueeze(-2)
    if not isinstance(t, _Tensor) or t.dim() != len(lead) + 2 or t.shape[-2] < 1 or D % t.shape[-2]:
        raise ValueError(f"{what}: {name} must be a tensor ({', '.join(map(str, lead))}, [G,] N) with G a divisor of D = {D}")
    return _seq(what, name, t, (*lead, t.shape[-2], N), dtype)


def _scan_args(what, x, dt, a, b, c, skip, gate, dt_bias, lead):
    """The checked operands; b and c with their group dimension."""
    D = x.shape[-1]
    if not isinstance(a, _Tensor) or a.dim() != 2 or a.shape[0] != D or not 1 <= a.shape[1] <= _lib.VSV_SSM_MAX_STATE or D < 1:
        raise ValueError(f"{what}: a must be a tensor (D, N) with 1 to {_lib.VSV_SSM_MAX_STATE} states")
    N = a.shape[1]
    x = _seq(what, "x", x, (*lead, D))
    dt = _seq(what, "dt", dt, (*lead, D), x.dtype)
    gate = None if gate is None else _seq(what, "gate", gate, (*lead, D), x.dtype)
    b, c = _grouped(what, "b", b, lead, D, N, x.dtype), _grouped(what, "c", c, lead, D, N, x.dtype)
    if b.shape != c.shape:
        raise ValueError(f"{what}: b has {b.shape[-2]} groups and c {c.shape[-2]}")
    a, skip, dt_bias = _f32(what, "a", a, (D, N)), _f32(what, "skip", skip, (D,)), _f32(what, "dt_bias", dt_bias, (D,))
    return x, dt, a, b, c, skip, gate, dt_bias


def ssm_scan(x, dt, a, b, c, skip=None, gate=None, *, dt_bias=None, softplus=True, initial_state=None, lengths=None,
             return_state=False):
    """The selective scan over whole sequences: x, dt [, gate] (B, T, D), a (D, N) with 1 to 16 states (negative where the
    state is to decay), b, c (B, T, [G,] N), skip, dt_bias (D).  softplus=False takes dt + dt_bias as the time step itself.
    initial_state (B, D, N).  Returns y (B, T, D) [, the state behind the last step (B, D, N) in float32].

    For gradients the states before every eighth step are kept (in float32: N / 2 bytes per element of x, N rounded up to
    4, 8 or 16).  A training step captured into a HIP graph wants parameters without a live eager graph of their own, as any
    captured backward pass of torch's does."""
    what = "ssm_scan"
    if not isinstance(x, _Tensor) or x.dim() != 3:
        raise ValueError(f"{what}: x must be a tensor (B, T, D)")
    B, T, D = x.shape
    x, dt, a, b, c, skip, gate, dt_bias = _scan_args(what, x, dt, a, b, c, skip, gate, dt_bias, (B, T))
    initial_state = _f32(what, "initial_state", initial_state, (B, D, a.shape[1]))
    lengths = _lengths(what, lengths, B)
    _same_gpu(what, x, dt, a, b, c, skip, gate, dt_bias, initial_state, lengths)
    if _wants_grad(x, dt, a, b, c, skip, gate, dt_bias, initial_state):
        from .autograd import SsmScan
        y, state = SsmScan.apply(x, dt, a, b, c, skip, gate, dt_bias, initial_state, lengths, bool(softplus), bool(return_state))
    else:
        y, state, _, _ = scan_forward(x, dt, a, b, c, skip, gate, dt_bias, initial_state, lengths, bool(softplus), return_state, False)
    return (y, state) if return_state else y


def _scan_desc(x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, softplus, B, T, y, state):
    D, N = a.shape
    if T is not None:
        x_bs, x_ts, _ = x.stride()
        dt_bs, dt_ts, _ = dt.stride()
        g_bs, g_ts, _ = gate.stride() if gate is not None else (0, 0, 0)
        b_bs, b_ts, b_gs, _ = b.stride()
        c_bs, c_ts, c_gs, _ = c.stride()
    else:                                                                  # (B, D) rows: one step, no time stride
        T = 1
        x_bs, x_ts, dt_bs, dt_ts, b_ts, c_ts, g_ts = x.stride(0), 0, dt.stride(0), 0, 0, 0, 0
        g_bs = gate.stride(0) if gate is not None else 0
        b_bs, b_gs, _ = b.stride()
        c_bs, c_gs, _ = c.stride()
    return _lib.VsvSsm(_TYPES[x.dtype], N, softplus, B, T, D, b.shape[-2], x.data_ptr(), x_bs, x_ts, dt.data_ptr(), dt_bs, dt_ts,
                       _ptr(gate), g_bs, g_ts, b.data_ptr(), b_bs, b_ts, b_gs, c.data_ptr(), c_bs, c_ts, c_gs,
                       a.data_ptr(), _ptr(skip), _ptr(dt_bias), _ptr(state_in), _ptr(lengths), y.data_ptr(), _ptr(state), None)


def scan_forward(x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, softplus, want_state, save):
    """The launches behind ssm_scan: (y, state | None, the descriptor vsv_ssm_scan_backward takes again, saved | None)."""
    (B, T, D), N = x.shape, a.shape[1]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    state = torch.empty((B, D, N), dtype=torch.float32, device=x.device) if want_state else None
    d = _scan_desc(x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, softplus, B, T, y, state)
    ref = C.byref(d)
    saved = None
    if save:
        saved = torch.empty(_size("vsv_ssm_saved_floats", ref), dtype=torch.float32, device=x.device)
        d.saved = saved.data_ptr() or None
    nbytes = _size("vsv_ssm_scan_ws_bytes", ref)
    ws = _workspace(nbytes, x.device) if nbytes else None
    _call("vsv_ssm_scan", x.get_device(), ref, _ptr(ws), nbytes)
    return y, state, d, saved


def ssm_step(x, dt, a, b, c, skip=None, gate=None, *, state, dt_bias=None, softplus=True):
    """ssm_scan for one new token of every row: x, dt [, gate] (B, D), b, c (B, [G,] N) -> y (B, D); state (B, D, N),
    contiguous float32, is updated in place.  No gradients."""
    what = "ssm_step"
    if not isinstance(x, _Tensor) or x.dim() != 2:
        raise ValueError(f"{what}: x must be a tensor (B, D)")
    B, D = x.shape
    x, dt, a, b, c, skip, gate, dt_bias = _scan_args(what, x, dt, a, b, c, skip, gate, dt_bias, (B,))
    _in_place(what, state, (B, D, a.shape[1]))
    _same_gpu(what, x, dt, a, b, c, skip, gate, dt_bias, state)
    if _wants_grad(x, dt, a, b, c, skip, gate, dt_bias, state):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    d = _scan_desc(x, dt, a, b, c, skip, gate, dt_bias, None, None, bool(softplus), B, None, y, state)
    _call("vsv_ssm_step", x.get_device(), C.byref(d))
    _touched(state)
    return y


# ---- the memory they make up -------------------------------------------------------------------------------------

class SsmMemory(torch.nn.Module):
    """A sequence memory called as nn.LSTM(batch_first=True) is: forward(x (B, T, input_size), state=None, lengths=None) ->
    (y (B, T, hidden_size), state), state = (the convolution's (B, taps - 1, hidden_size), the scan's
    (B, hidden_size, state_size)).  step(x (B, input_size), state) takes one new token and updates the state in place."""

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
        x, gate = self.in_proj(x).chunk(2, dim=-1)
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
