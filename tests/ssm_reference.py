"""Plain 64-bit forms of vsv.ssm's operators, step by step and with their gradients' formulas, on the CPU.

absolute=True returns, for every output, the sum of the absolute values of the terms that make it up: what a rounding error
in 32 bits is relative to.
"""
import torch


def _d(t):
    return None if t is None else t.detach().double().cpu()


def _silu(v, absolute):
    s = torch.sigmoid(v)
    if absolute:                          # (the slope s + s v (1 - s) has two terms, which cancel around v = -1.28)
        return (v * s).abs(), s * (1 + v.abs() * (1 - s))
    return v * s, s * (1 + v * (1 - s))


def conv_ref(x, w, bias, h0, lengths, silu, dy=None, dh=None, absolute=False):
    x, w, bias, h0, dy, dh = map(_d, (x, w, bias, h0, dy, dh))
    (B, T, D), K = x.shape, w.shape[1]
    ends = [T] * B if lengths is None else [min(max(int(n), 0), T) for n in lengths]
    mag = (lambda t: t.abs()) if absolute else (lambda t: t)
    bias = torch.zeros(D).double() if bias is None else bias
    out = {"y": torch.zeros(B, T, D).double(), "state": torch.zeros(B, K - 1, D).double(), "x": torch.zeros(B, T, D).double(),
           "w": torch.zeros(D, K).double(), "bias": torch.zeros(D).double(), "h0": torch.zeros(B, K - 1, D).double()}
    for i, n in enumerate(ends):
        xs = torch.cat([torch.zeros(K - 1, D).double() if h0 is None else h0[i], x[i, :n]], 0)
        out["state"][i] = xs[n:]
        pre = bias + sum(xs[k:k + n] * w[:, k] for k in range(K))
        size = mag(bias) + sum(mag(xs[k:k + n] * w[:, k]) for k in range(K))
        act, slope = _silu(pre, absolute) if silu else (mag(pre), torch.ones_like(pre))
        out["y"][i, :n] = act + (size if absolute else 0)
        d_xs = torch.zeros_like(xs)
        if dh is not None:
            d_xs[n:] += mag(dh[i])
        if dy is not None:
            ds = mag(dy[i, :n]) * slope + (mag(dy[i, :n]) * size if absolute else 0)     # (the slope's own error: |act''| <= 1/2 of pre's)
            for k in range(K):
                d_xs[k:k + n] += ds * mag(w[:, k])
                out["w"][:, k] += (ds * mag(xs[k:k + n])).sum(0)
            out["bias"] += ds.sum(0)
        out["h0"][i], out["x"][i, :n] = d_xs[:K - 1], d_xs[K - 1:]
    return out


def scan_ref(x, dt, a, b, c, skip, gate, dt_bias, h0, lengths, softplus=True, dy=None, dh=None, absolute=False):
    """b, c (B, T, G, N).  Outputs y, state and, for the gradients, the arguments' names."""
    x, dt, a, b, c, skip, gate, dt_bias, h0, dy, dh = map(_d, (x, dt, a, b, c, skip, gate, dt_bias, h0, dy, dh))
    (B, T, D), N, G = x.shape, a.shape[1], b.shape[2]
    group = torch.arange(D) // (D // G)
    mag = (lambda t: t.abs()) if absolute else (lambda t: t)
    skip = torch.zeros(D).double() if skip is None else skip
    raw = dt + (0 if dt_bias is None else dt_bias)
    delta = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    live = torch.ones(B, T).double() if lengths is None else torch.stack(
        [(torch.arange(T) < int(n)).double() for n in lengths])
    x, dy = torch.where(live[:, :, None] > 0, x, 0.0), None if dy is None else torch.where(live[:, :, None] > 0, dy, 0.0)
    delta = torch.where(live[:, :, None] > 0, delta, 0.0)
    slope = torch.where(live[:, :, None] > 0, slope, 0.0)
    b, c = (torch.where(live[:, :, None, None] > 0, t, 0.0) for t in (b, c))
    if gate is not None:
        gate = torch.where(live[:, :, None] > 0, gate, 0.0)
        act, dact = _silu(gate, absolute)
    else:
        act = dact = torch.ones_like(x)
    x, b, c, skip = mag(x), mag(b), mag(c), mag(skip)
    A, am = a, mag(a)
    dm = mag(delta)
    h = torch.zeros(B, D, N).double() if h0 is None else mag(h0)
    hs, y = [h], torch.zeros(B, T, D).double()
    for t in range(T):
        h = torch.exp(delta[:, t, :, None] * A) * h + (dm[:, t] * x[:, t])[:, :, None] * b[:, t][:, group]
        hs.append(h)
        y[:, t] = (h * c[:, t][:, group]).sum(-1) + skip * x[:, t]
    out = {"y": y * act, "state": h}
    if dy is None and dh is None:
        return out
    dy = torch.zeros_like(x) if dy is None else mag(dy)
    q = torch.zeros(B, D, N).double() if dh is None else mag(dh)
    g = dy * act
    out |= {"x": torch.zeros_like(x), "dt": torch.zeros_like(x), "a": torch.zeros_like(a), "b": torch.zeros_like(b),
            "c": torch.zeros_like(c), "skip": (g * x).sum((0, 1)), "gate": dy * y * dact}
    onto = torch.zeros(G, D).double()
    onto[group, torch.arange(D)] = 1
    for t in reversed(range(T)):
        decay = torch.exp(delta[:, t, :, None] * A)
        bt, ct = b[:, t][:, group], c[:, t][:, group]
        q = q + ct * g[:, t, :, None]
        out["c"][:, t] = onto @ (hs[t + 1] * g[:, t, :, None])
        out["b"][:, t] = onto @ (q * (dm[:, t] * x[:, t])[:, :, None])
        w = q * decay * hs[t]
        out["a"] += (w * dm[:, t, :, None]).sum(0)
        qb = (q * bt).sum(-1)
        out["x"][:, t] = qb * dm[:, t] + g[:, t] * skip
        out["dt"][:, t] = ((w * am).sum(-1) + qb * x[:, t]) * slope[:, t]
        q = q * decay
    out |= {"h0": q, "dt_bias": out["dt"].sum((0, 1))}
    return out


def scan_plan(B, T, D, N, G, forward=True):
    """(lanes that share a channel, segments, whether a launch of its own joins them) of a scan: the launcher's rule, with which
    kernels a size runs.  One lane: ssm_ends_kernel and ssm_scan_kernel, more: ssm_shared_kernel; joined: ssm_join_kernel."""
    R = 4 if N <= 4 else 8 if N <= 8 else 16
    waves, tiles, S, P = B * G * -(-(D // G) // 64), -(-T // 8), 1, 1
    if 0 < waves < 512:
        if forward and N > 4 and (T < 64 or waves * tiles <= 6144):
            P = R // 4
        if T >= (64 if P > 1 else 40):
            S = min(-(-2048 // (waves * P)), tiles // 2, 256)
    S = -(-tiles // -(-tiles // S)) if tiles else 1
    return P, S, S >= 24


# (B, T, D, N, G) -> what of it: every way that a forward pass of 5 to 16 states is divided, for either padded number of states
SCAN_PLANS = {
    (7, 41, 70, 16, 1): "shared", (7, 41, 70, 8, 1): "shared",
    (60, 130, 40, 13, 1): "shared split", (60, 130, 40, 6, 2): "shared split",
    (3, 700, 66, 16, 1): "shared joined", (3, 700, 66, 8, 2): "shared joined",
    (520, 20, 40, 16, 1): "alone", (260, 21, 130, 13, 1): "alone", (520, 20, 40, 8, 1): "alone", (515, 75, 24, 9, 2): "alone",
    (400, 131, 24, 16, 1): "alone split", (200, 250, 70, 5, 1): "alone split",
    (80, 620, 24, 16, 1): "alone joined", (40, 617, 70, 11, 1): "alone joined", (40, 620, 70, 8, 1): "alone joined",
}


def check(name, got, want, size, k):
    """|got - want| <= half a step of got's type at want + k half steps of float32 at the terms' size."""
    got, dtype = got.detach(), got.dtype
    assert tuple(got.shape) == tuple(want.shape), (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    err = (got.double().cpu() - want).abs()
    tiny = torch.finfo(dtype).smallest_normal
    bound = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + k * 2.0 ** -24 * size + tiny
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound (largest error {err.max().item():.3g})"
