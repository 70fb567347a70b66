"""AdamW over many tensors in one launch, with moments in 32 bits or in 8 (vsv_adamw_multi).

Beside torch.optim.AdamW, which CVAEMemRand.train_step turns into vsv_adamw_step (float32 parameters whose gradients are one
flat buffer), this optimizer takes any contiguous float32 / bfloat16 / float16 parameters with gradients of their own, and can
hold both moments in 8 bits: 2.03 bytes a parameter instead of 8.  It works wherever a torch optimizer does -- schedulers,
parameter groups, state_dict, and the model classes' train_step(x, optimizer).
"""
from __future__ import annotations

import array

import torch

from . import lib as _lib
from .ssm import _TYPES, _call, _touched


class AdamW(torch.optim.Optimizer):
    """AdamW(params, lr, betas, eps, weight_decay, state_bits=32 | 8): decoupled weight decay, bias-corrected moments.

    state_bits=8: per block of 256 elements a float32 scale of each moment; codes are rounded with a dither that is spread
    evenly over the steps, so small changes of the second moment are not lost.  An element whose gradient is not finite
    becomes NaN and keeps its moments (with 32 bits its moments follow the gradient).  The state of a parameter is
    {"step", "exp_avg", "exp_avg_sq"[, "exp_avg_scale", "exp_avg_sq_scale"]}; moments() gives the values in float32.

    The step count is a launch argument, so step() refuses to be captured into a HIP graph."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits!r}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    @property
    def state_bits(self):
        return self.defaults["state_bits"]                                 # (kept there, so copies and pickles have it)

    def add_param_group(self, group):
        super().add_param_group(group)
        try:
            g = self.param_groups[-1]
            lr, (b1, b2), eps, wd = float(g["lr"]), g["betas"], g["eps"], g["weight_decay"]
            if not (lr >= 0.0 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and wd >= 0.0):
                raise ValueError(f"AdamW: bad hyper-parameters lr={lr} betas={g['betas']} eps={eps} weight_decay={wd}")
            if g["state_bits"] != self.state_bits:
                raise ValueError("AdamW: all groups hold their moments in the same number of bits")
            for p in g["params"]:
                _check_param(p)
        except Exception:
            self.param_groups.pop()
            raise

    def _layout(self, p):
        """name -> (shape, type) of a parameter's state tensors."""
        if self.state_bits == 32:
            return {"exp_avg": (p.shape, torch.float32), "exp_avg_sq": (p.shape, torch.float32)}
        blocks = (-(-p.numel() // _lib.VSV_ADAMW_BLOCK),)
        return {"exp_avg": (p.shape, torch.int8), "exp_avg_sq": (p.shape, torch.uint8),
                "exp_avg_scale": (blocks, torch.float32), "exp_avg_sq_scale": (blocks, torch.float32)}

    def _init_state(self, p):
        self.state[p] = {"step": 0, **{k: torch.zeros(shape, dtype=dtype, device=p.device) for k, (shape, dtype) in self._layout(p).items()}}
        return self.state[p]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        state, calls = self.state, []
        for group in self.param_groups:                                    # everything is checked before anything is launched
            rows = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if p.dtype not in _TYPES or not p.is_contiguous():
                    _check_param(p)
                if g.layout is not torch.strided or g.dtype is not p.dtype or g.get_device() != p.get_device() or g.shape != p.shape:
                    raise ValueError("AdamW: a gradient needs its parameter's type, device and shape, and no sparse layout")
                if not p.is_cuda:
                    raise RuntimeError("AdamW: parameters must be on a GPU; there is no CPU fallback")
                st = state[p] or self._init_state(p)
                m = st["exp_avg"]
                if m.shape != p.shape or m.get_device() != p.get_device():
                    raise ValueError("AdamW: a parameter has changed its shape or device since its state was made")
                rows.setdefault((p.dtype, p.get_device(), st["step"]), []).append((p, g if g.is_contiguous() else g.contiguous(), st))
            calls += [(group, *key, rows[key]) for key in rows]
        if calls and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step cannot be captured into a HIP graph: the step count is a launch argument")
        for group, dtype, at, step, rows in calls:
            table = _table(rows, self.state_bits)
            b1, b2 = group["betas"]
            _call("vsv_adamw_multi", at, table.buffer_info()[0], len(rows), _TYPES[dtype], self.state_bits, float(group["lr"]),
                  float(b1), float(b2), float(group["eps"]), float(group["weight_decay"]), step + 1)
            written = []
            for p, _, st in rows:
                st["step"] = step + 1
                written += (p, st["exp_avg"], st["exp_avg_sq"])
            _touched(written)
        return loss

    @torch.no_grad()
    def moments(self):
        """([exp_avg], [exp_avg_sq]) in float32 of the parameters that have been stepped, in the groups' order: the state's own
        tensors with 32 bits, the values that the codes stand for with 8."""
        states = [st for st in (self.state.get(p) for g in self.param_groups for p in g["params"]) if st]
        if self.state_bits == 32:
            return [st["exp_avg"] for st in states], [st["exp_avg_sq"] for st in states]
        ms = [torch.empty_like(st["exp_avg"], dtype=torch.float32) for st in states]
        vs = [torch.empty_like(m) for m in ms]
        rows = {}
        for m, v, st in zip(ms, vs, states):
            rows.setdefault(m.get_device(), []).append((m, v, st))
        for at, part in rows.items():
            table = _table(part, 8)
            _call("vsv_adamw_read8", at, table.buffer_info()[0], len(part))
        return ms, vs

    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep their own types (torch's casts floating state to the parameter's), and nothing that
        does not fit the parameters is taken."""
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        if any(g.get("state_bits", self.state_bits) != self.state_bits for g in state_dict["param_groups"]):
            raise ValueError(f"AdamW: the saved moments are not held in {self.state_bits} bits")
        for i, p in zip(saved, params):
            st = state_dict["state"].get(i)
            if st and set(st) != {"step", *self._layout(p)}:
                raise ValueError(f"AdamW: the saved moments are not held in {self.state_bits} bits")
            for k, (shape, dtype) in self._layout(p).items() if st else ():
                if tuple(st[k].shape) != tuple(shape) or st[k].dtype != dtype:
                    raise ValueError(f"AdamW: saved {k} is {st[k].dtype} {tuple(st[k].shape)}, not {dtype} {tuple(shape)}")
        super().load_state_dict(state_dict)
        for i, p in zip(saved, params):
            if state_dict["state"].get(i):
                self.state[p] = {k: v.detach().to(device=p.device, copy=True).contiguous() if torch.is_tensor(v) else int(v)
                                 for k, v in state_dict["state"][i].items()}


def _check_param(p):
    if p.dtype not in _TYPES:
        raise ValueError(f"AdamW: parameters must be float32, bfloat16 or float16, not {p.dtype}")
    if not p.is_contiguous():
        raise ValueError("AdamW: parameters must be contiguous")


def _table(rows, bits):
    """struct vsv_adamw_tensor[len(rows)] of (p, g, state) rows, as 64-bit words."""
    words = []
    for p, g, st in rows:
        m = st["exp_avg"]
        if bits == 8:
            words += (p.data_ptr(), g.data_ptr(), m.data_ptr(), st["exp_avg_sq"].data_ptr(), st["exp_avg_scale"].data_ptr(),
                      st["exp_avg_sq_scale"].data_ptr(), m.numel())
        else:
            words += (p.data_ptr(), g.data_ptr(), m.data_ptr(), st["exp_avg_sq"].data_ptr(), 0, 0, m.numel())
    return array.array("Q", words)
