"""torch.autograd.Function over the HIP forward / backward kernels.

The reference's forward() (vae/cvae_with_mem_randomized.py:1022-1074) returns tensors that carry an
autograd graph, so callers may write their own loss and call .backward() instead of train_step().
CVAEForward gives the HIP path the same property: forward = TrainEngine.forward_saved (the three
vsv_train_* launches, activations kept on the device), backward = TrainEngine.backward_saved (decoder
head, BPTT, conv backward kernels) from whatever gradients autograd hands back for the five outputs,
scattered onto the nn.Parameters through the packing index maps.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import lib as vlib, ssm


class CVAEForward(torch.autograd.Function):
    """apply(te, surf, ex | None, horizon, eps | None, seed, dropout_p, dropout_seed, *params)
    -> (recon (B,H,Q,5,5), ex_recon (B,H,X) or an empty tensor, z_mean, z_log_var, z), float32.
    `params` are the model's parameters in the order the TrainEngine was built with; the engine's
    packed blob must have been refreshed from them (CVAEMemRand._engine does)."""

    @staticmethod
    def forward(ctx, te, surf, ex, horizon, eps, seed, dropout_p, dropout_seed, *params):
        c = te.forward_saved(surf, ex, int(horizon), eps, int(seed), float(dropout_p), int(dropout_seed))
        ctx.te, ctx.c = te, c
        ctx.want_dsurf = bool(ctx.needs_input_grad[1])
        ctx.surf_meta = (surf.shape, surf.dtype, surf.device)
        ctx.param_meta = [(p.dtype, p.device) for p in params]
        o = c.outputs
        e = o["ex"] if o["ex"] is not None else torch.empty(0, device=te.dev)
        if o["ex"] is None:
            ctx.mark_non_differentiable(e)
        return o["surf"], e, o["z_mean"], o["z_log_var"], o["z"]

    @staticmethod
    def backward(ctx, d_s, d_e, d_zm, d_zl, d_z):
        te, c = ctx.te, ctx.c
        if c is None:
            raise RuntimeError("CVAEForward: backward through the HIP path a second time (the saved "
                               "activations are freed after the first backward, as with retain_graph=False)")
        ctx.c = None
        if d_s is None:
            d_s = torch.zeros_like(c.outputs["surf"])
        if c.outputs["ex"] is None:
            d_e = None
        gp = te.backward_saved(c, d_s, d_e, d_zm, d_zl, d_z, ctx.want_dsurf)
        grads = []
        for g, (dt, dev), need in zip(te.param_grads(gp), ctx.param_meta, ctx.needs_input_grad[8:]):
            grads.append(g.to(device=dev, dtype=dt) if need else None)
        d_surf = None
        if ctx.want_dsurf:
            shape, dt, dev = ctx.surf_meta
            d_surf = c.outputs["d_surface"].reshape(shape).to(device=dev, dtype=dt)
        return (None, d_surf, None, None, None, None, None, None, *grads)


class ShortConv(torch.autograd.Function):
    """vsv.ssm.short_conv's gradient: apply(x, weight, bias | None, initial_state | None, lengths | None, silu, want_state) ->
    (y, state | None).  The backward pass computes the pre-activation again from x, so only the inputs are kept."""

    @staticmethod
    def forward(ctx, x, weight, bias, state_in, lengths, silu, want_state):
        y, state, _ = ssm.conv_forward(x, weight, bias, state_in, lengths, silu, want_state)
        ctx.save_for_backward(x, weight, bias, state_in, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_state):
        x, weight, bias, state_in, lengths = ctx.saved_tensors
        if dy is None and d_state is None:
            return (None,) * 7
        (B, T, D), K = x.shape, weight.shape[1]
        dy = torch.zeros_like(x) if dy is None else ssm._last(dy)
        d_state = None if d_state is None else d_state.contiguous()
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        need = ctx.needs_input_grad
        dw = torch.empty_like(weight) if need[1] else None
        db = torch.empty_like(bias) if bias is not None and need[2] else None
        ds = torch.empty_like(state_in) if state_in is not None and need[3] else None
        d = vlib.VsvShortConv(ssm._TYPES[x.dtype], K, int(ctx.silu), B, T, D, x.data_ptr(), x.stride(0), x.stride(1),
                              weight.data_ptr(), ssm._ptr(bias), ssm._ptr(state_in), ssm._ptr(lengths), dx.data_ptr(), None)
        g = vlib.VsvShortConvGrads(dy.data_ptr(), dy.stride(0), dy.stride(1), ssm._ptr(d_state), dx.data_ptr(), ssm._ptr(dw), ssm._ptr(db),
                                   ssm._ptr(ds))
        nbytes = ssm._size("vsv_short_conv_backward_ws_bytes", C.byref(d))
        ws = ssm._workspace(nbytes, x.device)
        ssm._call("vsv_short_conv_backward", x.get_device(), C.byref(d), C.byref(g), ws.data_ptr(), nbytes)
        return dx if need[0] else None, dw, db, ds, None, None, None


class SsmScan(torch.autograd.Function):
    """vsv.ssm.ssm_scan's gradient: apply(x, dt, a, b, c, skip | None, gate | None, dt_bias | None, initial_state | None,
    lengths | None, softplus, want_state) -> (y, state | None).  Kept: the inputs and the states before every eighth step."""

    @staticmethod
    def forward(ctx, x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, softplus, want_state):
        y, state, _, saved = ssm.scan_forward(x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, softplus, want_state, True)
        ctx.save_for_backward(x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, saved)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_state):
        x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, saved = ctx.saved_tensors
        if dy is None and d_state is None:
            return (None,) * 12
        (B, T, D), need = x.shape, ctx.needs_input_grad
        dy = torch.zeros_like(x) if dy is None else ssm._last(dy)
        d_state = None if d_state is None else d_state.contiguous()
        whole = torch.contiguous_format
        dx, ddt = torch.empty_like(x, memory_format=whole), torch.empty_like(x, memory_format=whole)
        dgate = torch.empty_like(x, memory_format=whole) if gate is not None else None
        db, dc = torch.empty_like(b, memory_format=whole), torch.empty_like(c, memory_format=whole)
        like = lambda t, k: torch.empty_like(t) if t is not None and need[k] else None        # noqa: E731
        da, dskip, ddt_bias, ds = like(a, 2), like(skip, 5), like(dt_bias, 7), like(state_in, 8)
        d = ssm._scan_desc(x, dt, a, b, c, skip, gate, dt_bias, state_in, lengths, ctx.softplus, B, T, dx, None)
        d.saved = saved.data_ptr() or None
        g = vlib.VsvSsmGrads(dy.data_ptr(), dy.stride(0), dy.stride(1), ssm._ptr(d_state), dx.data_ptr(), ddt.data_ptr(), ssm._ptr(dgate),
                             db.data_ptr(), dc.data_ptr(), ssm._ptr(da), ssm._ptr(dskip), ssm._ptr(ddt_bias), ssm._ptr(ds))
        ref = C.byref(d)
        nbytes = ssm._size("vsv_ssm_scan_backward_ws_bytes", ref)
        ws = ssm._workspace(nbytes, x.device)
        ssm._call("vsv_ssm_scan_backward", x.get_device(), ref, C.byref(g), ws.data_ptr(), nbytes)
        pick = lambda t, k: t if need[k] else None                                             # noqa: E731
        return (pick(dx, 0), pick(ddt, 1), da, pick(db, 3), pick(dc, 4), dskip, pick(dgate, 6), ddt_bias, ds, None, None, None)
