"""AdamW over many tensors in one launch, with moments in 32 bits or in 8 (vsv_adamw_multi).

Beside torch.optim.AdamW, which CVAEMemRand.train_step turns into vsv_adamw_step (float32 parameters whose gradients are one
flat buffer), this optimizer takes any contiguous float32 / bfloat16 / float16 parameters with gradients of their own, and can
hold both moments in 8 bits: 2.03 bytes a parameter instead of 8.  It works wherever a torch optimizer does -- schedulers,
parameter groups, state_dict, and the model classes' train_step(x, optimizer).
"""
from __future__ import annotations

import torch

from . import lib as _lib
from . import native as _native


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
            _check_options(g)
            if len(set(map(id, g["params"]))) < len(g["params"]):
                raise ValueError("AdamW: a parameter is in its group twice")
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
        if p.is_cuda:                                                      # (under capture the zeros would only be recorded)
            with torch.cuda.device(p.device):
                _native.load().refuse_capture()
        self.state[p] = {"step": 0, **{k: torch.zeros(shape, dtype=dtype, device=p.device) for k, (shape, dtype) in self._layout(p).items()}}
        return self.state[p]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        state, calls, states = self.state, [], []
        wide = self.state_bits == 32
        for group in self.param_groups:
            rows = {}
            for p in group["params"]:
                g = p.grad
                if g is not None:
                    st = state.get(p) or self._init_state(p)
                    rows.setdefault(st["step"], []).append((p, g, st))
            b1, b2 = group["betas"]
            for step, part in rows.items():
                ps, gs, sts = zip(*part)
                calls.append((ps, gs, [st["exp_avg"] for st in sts], [st["exp_avg_sq"] for st in sts],
                              [] if wide else [st["exp_avg_scale"] for st in sts], [] if wide else [st["exp_avg_sq_scale"] for st in sts],
                              float(group["lr"]), float(b1), float(b2), float(group["eps"]), float(group["weight_decay"]), step + 1))
                states += sts
        if calls:
            _native.load().adamw_step(self.state_bits, calls)              # (checks everything before it launches anything)
            for st in states:
                st["step"] += 1
        return loss

    @torch.no_grad()
    def moments(self):
        """([exp_avg], [exp_avg_sq]) in float32 of the parameters that have been stepped, in the groups' order: the state's own
        tensors with 32 bits, the values that the codes stand for with 8."""
        states = [st for st in (self.state.get(p) for g in self.param_groups for p in g["params"]) if st]
        m, v = [st["exp_avg"] for st in states], [st["exp_avg_sq"] for st in states]
        if self.state_bits == 32:
            return m, v
        return _native.load().adamw_read8(m, v, [st["exp_avg_scale"] for st in states], [st["exp_avg_sq_scale"] for st in states])

    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep their own types (torch's casts floating state to the parameter's), and nothing that
        does not fit the parameters is taken.  Hooks see and change what they do of torch's."""
        given = []
        hooks = [self.register_load_state_dict_pre_hook(lambda _, d: given.append(self._fitting(d))),      # (behind every other)
                 self.register_load_state_dict_post_hook(lambda _: self._take(given[0]), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _fitting(self, state_dict):
        """[(parameter, its saved state or None)], refused where it does not fit."""
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        if any(g.get("state_bits", self.state_bits) != self.state_bits for g in state_dict["param_groups"]):
            raise ValueError(f"AdamW: the saved moments are not held in {self.state_bits} bits")
        for g in state_dict["param_groups"]:
            _check_options(g)
        rows = [(p, state_dict["state"].get(i)) for i, p in zip(saved, params)]
        for p, st in rows:
            if st and set(st) != {"step", *self._layout(p)}:
                raise ValueError(f"AdamW: the saved moments are not held in {self.state_bits} bits")
            for k, (shape, dtype) in self._layout(p).items() if st else ():
                if tuple(st[k].shape) != tuple(shape) or st[k].dtype != dtype:
                    raise ValueError(f"AdamW: saved {k} is {st[k].dtype} {tuple(st[k].shape)}, not {dtype} {tuple(shape)}")
        return rows

    def _take(self, rows):
        for p, st in rows:
            if st:
                # (torch's own optimizers keep the step count in a tensor: here it groups the parameters, and is a launch argument)
                self.state[p] = {k: int(v) if k == "step" else v.detach().to(device=p.device, copy=True).contiguous()
                                 for k, v in st.items()}


def _check_options(group):
    """Options of torch's Adam family that a group, or a state saved by one of them, may carry and this step does not have."""
    if group.get("amsgrad") or group.get("maximize") or (group.get("decoupled_weight_decay") is False and group["weight_decay"]):
        raise ValueError("AdamW: amsgrad, maximize and coupled weight decay are not built")


def _check_param(p):
    if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"AdamW: parameters must be float32, bfloat16 or float16, not {p.dtype}")
    if not p.is_contiguous() or p.is_neg():                                # (a negative view's memory holds the values' opposites)
        raise ValueError("AdamW: parameters must be contiguous, and no negative views")
