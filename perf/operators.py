"""The sequence-memory and optimizer operators as measured work.

Four operators, each as one pass of a user's program:

  scan   the selective state space scan over whole sequences: a prompt, or a training step's forward and backward
  conv   the short causal convolution in front of it: a prompt, or forward and backward
  step   both for one new token of every sequence, the states updated in place
  adamw  one optimizer step over many tensors, with moments in 32 bits or in 8

With ``own`` false ``run`` computes them in elementary torch operations in 32 bits (64 for what decides a code of
8 bits); with ``own`` true it calls the package's entry points.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}

LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2
BLOCK = 256                                   # elements that share a scale where moments are held in 8 bits
WEYL_I, WEYL_T = 0xC13FA9A9, 0x91E10DA5       # 2^32 / 1.32472 and 2^32 / 1.75488: the dither's steps


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed():
    return [
        # A training driver's context batch: 64 windows of 60 days, hidden width 100, before generation.
        {"name": "scan prompt 64x60x100", "op": "scan", "train": False, "B": 64, "T": 60, "D": 100, "N": 16, "G": 1,
         "dtype": "fp32", "ragged": False, "carry": True},
        # One long history read at once: everything has to come from splitting the time axis.
        {"name": "scan prompt 1x16384x2048", "op": "scan", "train": False, "B": 1, "T": 16384, "D": 2048, "N": 16, "G": 1,
         "dtype": "bf16", "ragged": False, "carry": True},
        # The same context batch as a training step: 60 days of context and 30 of horizon.
        {"name": "scan train 64x90x100", "op": "scan", "train": True, "B": 64, "T": 90, "D": 100, "N": 16, "G": 1,
         "dtype": "fp32", "ragged": False, "carry": False},
        # A padded batch of odd sizes with two groups, an odd state size and a state carried in from earlier windows.
        {"name": "scan train ragged 5x777x198", "op": "scan", "train": True, "B": 5, "T": 777, "D": 198, "N": 13, "G": 2,
         "dtype": "fp32", "ragged": True, "carry": True},
        # A wide memory in training.
        {"name": "scan train 4x2048x2048", "op": "scan", "train": True, "B": 4, "T": 2048, "D": 2048, "N": 16, "G": 1,
         "dtype": "bf16", "ragged": False, "carry": False},
        # The convolution in front of it: a padded prompt batch of an odd width, then a wide training step.
        {"name": "conv prompt ragged 16x333x515", "op": "conv", "train": False, "B": 16, "T": 333, "D": 515, "K": 3,
         "dtype": "fp32", "ragged": True, "carry": True},
        {"name": "conv train 8x2048x4096", "op": "conv", "train": True, "B": 8, "T": 2048, "D": 4096, "K": 4,
         "dtype": "bf16", "ragged": False, "carry": False},
        # Single tokens: one sequence, where the call itself counts, and a full batch of a thousand samples.
        {"name": "step 1x2048", "op": "step", "B": 1, "D": 2048, "N": 16, "G": 1, "K": 4, "dtype": "bf16"},
        {"name": "step 1000x4096", "op": "step", "B": 1000, "D": 4096, "N": 16, "G": 1, "K": 4, "dtype": "bf16"},
        # The optimizer: the surface encoder's own 18 tensors, then 168 M elements of a wide stack of layers.
        {"name": "adamw 8-bit encoder", "op": "adamw", "bits": 8, "layers": 0, "width": 100, "dtype": "fp32"},
        {"name": "adamw 32-bit 4x2048", "op": "adamw", "bits": 32, "layers": 4, "width": 2048, "dtype": "fp32"},
        {"name": "adamw 8-bit 4x2048", "op": "adamw", "bits": 8, "layers": 4, "width": 2048, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "conv", "conv", "step", "adamw", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "adamw":
        layers = rng.randint(0, 4)
        width = _log(rng, 16, 128) if layers == 0 else _log(rng, 64, 2048)
        return {"op": op, "bits": rng.choice([8, 32]), "layers": layers, "width": width, "dtype": dtype}
    if op == "step":
        B, D = _log(rng, 1, 1000), _log(rng, 64, 4096)
        G = rng.choice([1, 1, 2])
        return {"op": op, "B": B, "D": D - D % G, "N": rng.choice([16, 16, 8, rng.randint(1, 16)]), "G": G,
                "K": rng.choice([4, 4, 3, 2]), "dtype": dtype}
    train = rng.random() < 0.5
    D = _log(rng, 24, 4096)
    if rng.random() < 0.5:
        D = max(8, D - D % 8)
    T = _log(rng, 1, 16384)
    most = (16777216 if train else 33554432) if op == "scan" else 67108864
    B = _log(rng, 1, max(1, min(64, most // (T * D)))) if T * D <= most else 1
    T = max(1, min(T, most // (B * D)))
    case = {"op": op, "train": train, "B": B, "T": T, "D": D, "dtype": dtype, "ragged": rng.random() < 0.5,
            "carry": rng.random() < 0.5}
    if op == "conv":
        return {**case, "K": rng.choice([4, 4, 3, 2])}
    G = rng.choice([1, 1, 2])
    return {**case, "D": D - D % G, "N": rng.choice([16, 16, 8, rng.randint(1, 16)]), "G": G}


def _shapes(case):
    """The tensors of an adamw case: the surface encoder's for no layers, else `layers` layers of a wide stack."""
    w = case["width"]
    if case["layers"] == 0:
        conv = [(5, 1, 3, 3), (5,), (5, 5, 3, 3), (5,), (5, 5, 3, 3), (5,)]
        mem = [(4 * w, 128), (4 * w, w), (4 * w,), (4 * w,), (4 * w, w), (4 * w, w), (4 * w,), (4 * w,)]
        return conv + mem + [(12, w), (12,), (12, w), (12,)]
    return [(w, w), (w, w), (4 * w, w), (w, 4 * w), (w,)] * case["layers"]


# ---- the inputs --------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    f32 = torch.float32
    s = {"case": dict(case)}
    if case["op"] == "adamw":
        s["p"] = [normal(*sh, scale=0.05) for sh in _shapes(case)]
        # (gradients of a real step span orders of magnitude between tensors and within them)
        s["g"] = [(normal(*sh, scale=1e-3, dtype=f32) * torch.exp(2.0 * torch.randn(*sh, generator=gen, device=DEV))).to(dt)
                  for sh in _shapes(case)]
        s["step"] = 0
        return s
    B, D = case["B"], case["D"]
    if case["op"] in ("conv", "step"):
        s["w"] = normal(D, case["K"], scale=0.5, dtype=f32)
        s["wb"] = normal(D, scale=0.1, dtype=f32)
    if case["op"] in ("scan", "step"):
        N, G = case["N"], case["G"]
        s["a"] = -torch.arange(1, N + 1, device=DEV, dtype=f32) * (1.0 + 0.2 * uniform(D, N))
        s["skip"] = 1.0 + normal(D, scale=0.1, dtype=f32)
        step = torch.exp(math.log(1e-3) + uniform(D) * math.log(100.0))       # time steps of 0.001 to 0.1
        s["dt_bias"] = torch.log(torch.expm1(step))
    if case["op"] == "step":
        s["x"] = normal(B, D)
        s["dt"] = normal(B, D, scale=0.5)
        s["b"], s["c"], s["gate"] = normal(B, G, N), normal(B, G, N), normal(B, D)
        s["conv_state"] = normal(B, case["K"] - 1, D).to(f32)
        s["state"] = normal(B, D, N, scale=0.3, dtype=f32)
        return s
    T = case["T"]
    s["x"] = normal(B, T, D)
    if case["op"] == "scan":
        s["dt"] = normal(B, T, D, scale=0.5)
        s["b"], s["c"], s["gate"] = normal(B, T, G, N), normal(B, T, G, N), normal(B, T, D)
    s["h0"] = None
    if case["carry"]:
        s["h0"] = normal(B, D, N, scale=0.3, dtype=f32) if case["op"] == "scan" else normal(B, case["K"] - 1, D).to(f32)
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = (uniform(B) * (T + 1)).to(torch.int32).clamp_(max=T)
        s["lengths"][0] = T
    if case["train"]:
        s["dy"] = normal(B, T, D)
        s["dh"] = torch.randn(s["h0"].shape, generator=gen, device=DEV) if case["carry"] else None
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if own:
        return {"scan": _own_scan, "conv": _own_conv, "step": _own_step, "adamw": _own_adamw}[op](s)
    return {"scan": _plain_scan, "conv": _plain_conv, "step": _plain_step, "adamw": _plain_adamw}[op](s)


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vol-surface-vae-pub_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


def _own_scan(s):
    _package()
    from vsv.ssm import ssm_scan
    case = s["case"]
    names = ["x", "dt", "a", "b", "c", "skip", "gate", "dt_bias"] + (["h0"] if case["carry"] else [])
    if not case["train"]:
        return ssm_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], s["skip"], s["gate"], dt_bias=s["dt_bias"],
                        initial_state=s["h0"], lengths=s["lengths"], return_state=True)
    for n in names:
        s[n].requires_grad_(True)
    y, h = ssm_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], s["skip"], s["gate"], dt_bias=s["dt_bias"],
                    initial_state=s["h0"], lengths=s["lengths"], return_state=True)
    if case["carry"]:
        grads = torch.autograd.grad((y, h), [s[n] for n in names], (s["dy"], s["dh"]))
    else:
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y.detach(), "state": h.detach(), **{"d_" + n: g for n, g in zip(names, grads)}}


def _own_conv(s):
    _package()
    from vsv.ssm import short_conv
    case = s["case"]
    names = ["x", "w", "wb"] + (["h0"] if case["carry"] else [])
    if not case["train"]:
        return short_conv(s["x"], s["w"], s["wb"], initial_state=s["h0"], lengths=s["lengths"], return_state=True)
    for n in names:
        s[n].requires_grad_(True)
    y, h = short_conv(s["x"], s["w"], s["wb"], initial_state=s["h0"], lengths=s["lengths"], return_state=True)
    if case["carry"]:
        grads = torch.autograd.grad((y, h), [s[n] for n in names], (s["dy"], s["dh"]))
    else:
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y.detach(), "state": h.detach(), **{"d_" + n: g for n, g in zip(names, grads)}}


def _own_step(s):
    _package()
    from vsv.ssm import short_conv_step, ssm_step
    x = short_conv_step(s["x"], s["conv_state"], s["w"], s["wb"])
    y = ssm_step(x, s["dt"], s["a"], s["b"], s["c"], s["skip"], s["gate"], state=s["state"], dt_bias=s["dt_bias"])
    return {"x": x, "y": y, "conv_state": s["conv_state"], "state": s["state"]}


def _own_adamw(s):
    if "opt" not in s:
        _package()
        from vsv.optim import AdamW
        s["params"] = [torch.nn.Parameter(p) for p in s["p"]]
        for p, g in zip(s["params"], s["g"]):
            p.grad = g
        s["opt"] = AdamW(s["params"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=s["case"]["bits"])
    s["opt"].step()
    m, v = s["opt"].moments()
    return {"p": s["p"], "m": m, "v": v}


# ---- plain forms -------------------------------------------------------------------------------------------------

def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 from h = 0, by doubling: log2(T) passes over whole sequences."""
    T, step = a.shape[1], 1
    while step < T:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        if 2 * step < T:
            a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _per_channel(t, D):
    """(..., G, N) -> (..., D, N): every channel's row of its group."""
    return t.repeat_interleave(D // t.shape[-2], dim=-2)


def _valid(s, T):
    """(B, T, 1): 1 at the steps before a sequence's length."""
    if s["lengths"] is None:
        return None
    return (torch.arange(T, device=DEV)[None, :] < s["lengths"][:, None]).unsqueeze(-1)


def _plain_scan(s):
    case = s["case"]
    B, T, D, N = case["B"], case["T"], case["D"], case["N"]
    dtype = s["x"].dtype
    ok = _valid(s, T)
    x, dy_in = s["x"].detach().float(), None
    raw = s["dt"].detach().float() + s["dt_bias"].detach()
    delta = _softplus(raw)
    gate = s["gate"].detach().float()
    A, skip = s["a"].detach(), s["skip"].detach()
    b, c = _per_channel(s["b"].detach().float(), D), _per_channel(s["c"].detach().float(), D)
    if ok is not None:
        delta = torch.where(ok, delta, torch.zeros_like(delta))
    decay = torch.exp(delta.unsqueeze(-1) * A)                          # 1 behind a sequence's end
    h = (delta * x).unsqueeze(-1) * b
    if s["h0"] is not None:
        h[:, 0] += decay[:, 0] * s["h0"].detach()
    h = _recur(decay, h)
    y = (h * c).sum(-1) + skip * x
    sig = _sigmoid(gate)
    out = y * gate * sig
    last = h[:, T - 1].clone()
    if ok is not None:
        out = torch.where(ok, out, torch.zeros_like(out))
    if not case["train"]:
        return out.to(dtype), last
    dy = s["dy"].float()
    if ok is not None:
        dy = torch.where(ok, dy, torch.zeros_like(dy))
    d_gate = dy * y * sig * (1.0 + gate * (1.0 - sig))
    g = dy * gate * sig
    # the state's gradient runs backwards: q_t = c_t g_t + decay_{t+1} q_{t+1}
    q = g.unsqueeze(-1) * c
    if s["dh"] is not None:
        q[:, T - 1] += s["dh"]
    ahead = torch.cat([decay[:, 1:], torch.ones_like(decay[:, :1])], 1)
    q = _recur(ahead.flip(1), q.flip(1)).flip(1)
    del ahead
    G = case["G"]
    d_c = (g.unsqueeze(-1) * h).view(B, T, G, D // G, N).sum(3)
    d_b = ((delta * x).unsqueeze(-1) * q).view(B, T, G, D // G, N).sum(3)
    first = torch.zeros_like(h[:, :1]) if s["h0"] is None else s["h0"].detach().unsqueeze(1)
    w = q * decay * torch.cat([first, h[:, :-1]], 1)                     # gradient of the decay's exponent
    qb = (q * b).sum(-1)
    d_delta = (w * A).sum(-1) + qb * x
    d_a = (w * delta.unsqueeze(-1)).sum((0, 1))
    d_x = qb * delta + g * skip
    d_raw = d_delta * _sigmoid(raw)
    if ok is not None:
        d_raw = torch.where(ok, d_raw, torch.zeros_like(d_raw))
    got = {"y": out.to(dtype), "state": last, "d_x": d_x.to(dtype), "d_dt": d_raw.to(dtype), "d_a": d_a, "d_b": d_b.to(dtype),
           "d_c": d_c.to(dtype), "d_skip": (g * x).sum((0, 1)), "d_gate": d_gate.to(dtype), "d_dt_bias": d_raw.sum((0, 1))}
    if s["h0"] is not None:
        got["d_h0"] = q[:, 0] * decay[:, 0]
    return got


def _plain_conv(s):
    case = s["case"]
    B, T, D, K = case["B"], case["T"], case["D"], case["K"]
    dtype = s["x"].dtype
    ok = _valid(s, T)
    w, bias = s["w"].detach(), s["wb"].detach()
    before = s["h0"].detach() if s["h0"] is not None else torch.zeros(B, K - 1, D, device=DEV)
    xs = torch.cat([before, s["x"].detach().float()], 1)                  # (B, T + K - 1, D)
    rows = xs.unfold(1, T, 1)                                             # (B, K, D, T): tap k sees xs[k : k + T]
    pre = (rows * w.t()[None, :, :, None]).sum(1).transpose(1, 2) + bias
    sig = _sigmoid(pre)
    y = pre * sig
    if ok is None:
        last = xs[:, T:].clone()
    else:
        y = torch.where(ok, y, torch.zeros_like(y))
        at = s["lengths"].long()[:, None] + torch.arange(K - 1, device=DEV)
        last = xs.gather(1, at[:, :, None].expand(B, K - 1, D))
    if not case["train"]:
        return y.to(dtype), last
    dy = s["dy"].float()
    ds = dy * sig * (1.0 + pre * (1.0 - sig))
    if ok is not None:
        ds = torch.where(ok, ds, torch.zeros_like(ds))
    pad = torch.zeros(B, K - 1, D, device=DEV)
    # xs[j] feeds ds[j - k] through tap k
    at = torch.cat([pad, ds, pad], 1).unfold(1, T + K - 1, 1)             # (B, K, D, T + K - 1)
    d_xs = (at.flip(1) * w.t()[None, :, :, None]).sum(1).transpose(1, 2).contiguous()
    if s["dh"] is not None:
        if ok is None:
            d_xs[:, T:] += s["dh"]
        else:
            at = s["lengths"].long()[:, None] + torch.arange(K - 1, device=DEV)
            d_xs.scatter_add_(1, at[:, :, None].expand(B, K - 1, D), s["dh"])
    got = {"y": y.to(dtype), "state": last, "d_x": d_xs[:, K - 1:].to(dtype),
           "d_w": (rows * ds.transpose(1, 2).unsqueeze(1)).sum((0, 3)).t().contiguous(), "d_wb": ds.sum((0, 1))}
    if s["h0"] is not None:
        got["d_h0"] = d_xs[:, :K - 1].clone()
    return got


def _plain_step(s):
    case = s["case"]
    D = case["D"]
    dtype = s["x"].dtype
    xs = torch.cat([s["conv_state"], s["x"].float().unsqueeze(1)], 1)
    s["conv_state"].copy_(xs[:, 1:])
    pre = (xs * s["w"].t()).sum(1) + s["wb"]
    x_out = (pre * _sigmoid(pre)).to(dtype)
    x = x_out.float()                                                     # (the second call takes what the first returned)
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    h = s["state"] * torch.exp(delta.unsqueeze(-1) * s["a"]) + (delta * x).unsqueeze(-1) * _per_channel(s["b"].float(), D)
    s["state"].copy_(h)
    gate = s["gate"].float()
    y = ((h * _per_channel(s["c"].float(), D)).sum(-1) + s["skip"] * x) * gate * _sigmoid(gate)
    return {"x": x_out, "y": y.to(dtype), "conv_state": s["conv_state"], "state": s["state"]}


def _blocks(t):
    """A tensor's values as rows of BLOCK, the last one filled up with zeros."""
    flat = t.reshape(-1)
    fill = -flat.numel() % BLOCK
    return torch.cat([flat, flat.new_zeros(fill)]).view(-1, BLOCK) if fill else flat.view(-1, BLOCK)


def _encode(x, power, levels, scale, u):
    """Codes 0 .. levels of the values x in [0, scale] (64 bits), where code k stands for scale (k / levels)^power: of the two
    codes around a value the upper one where the value is more than a share u of the way."""
    full = float(levels) ** power
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)) * full, torch.zeros_like(x)).clamp_(max=full)
    k = torch.floor(torch.sqrt(y) if power == 2 else torch.sqrt(torch.sqrt(y)))
    k = k - (k ** power > y).double()
    k = k + ((k + 1.0) ** power <= y).double()
    below = k ** power
    return k + (y - below > u * ((k + 1.0) ** power - below)).double()


def _plain_adamw(s):
    bits = s["case"]["bits"]
    if "m" not in s:
        s["m"] = [torch.zeros(p.shape, device=DEV) for p in s["p"]]
        s["v"] = [torch.zeros(p.shape, device=DEV) for p in s["p"]]
    s["step"] += 1
    t = s["step"]
    rate = LR / (1.0 - BETA1 ** t)
    root = math.sqrt(1.0 - BETA2 ** t)
    for p, g, m, v in zip(s["p"], s["g"], s["m"], s["v"]):
        wide = torch.float64 if bits == 8 else torch.float32              # (a code of 8 bits is decided in 64)
        gw = g.to(wide)
        mw = m.to(wide) * BETA1 + gw * (1.0 - BETA1)
        vw = v.to(wide) * BETA2 + gw * gw * (1.0 - BETA2)
        p32 = p.detach().float() * (1.0 - LR * DECAY)
        p.copy_(p32 - rate * mw.float() / (torch.sqrt(vw.float()) / root + EPS))
        if bits == 8:
            index = _blocks(torch.arange(p.numel(), device=DEV))
            u = (((index * WEYL_I & 0xFFFFFFFF) + (t * WEYL_T & 0xFFFFFFFF) & 0xFFFFFFFF).double() + 0.5) * 2.0 ** -32
            mb, vb = _blocks(mw), _blocks(vw)
            ms, vs = mb.abs().amax(1, keepdim=True).float().double(), vb.amax(1, keepdim=True).float().double()
            km = _encode(mb.abs(), 2, 127, ms, u)
            kv = _encode(vb, 4, 255, vs, 1.0 - u)
            kv = torch.where((kv < 1) & (vb > 0) & (vs > 0), torch.ones_like(kv), kv)
            mw = (torch.sign(mb) * ms * (km / 127.0) ** 2).view(-1)[:p.numel()].view(p.shape)
            vw = (vs * (kv / 255.0) ** 4).view(-1)[:p.numel()].view(p.shape)
        m.copy_(mw)
        v.copy_(vw)
    return {"p": s["p"], "m": s["m"], "v": s["v"]}


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "adamw":
        n = sum(math.prod(sh) for sh in _shapes(case))
        if case["bits"] == 32:                                            # parameter and two moments both ways, the gradient in
            return {"bytes": n * (3 * e + 16), "flops": 14 * n}
        # (codes and scales both ways, and the moments once more as the values that they stand for)
        return {"bytes": n * (3 * e + 4 + 16 / BLOCK + 8), "flops": 40 * n}
    B, D = case["B"], case["D"]
    if case["op"] == "step":
        N, K = case["N"], case["K"]
        return {"bytes": B * D * (8 * N + 8 * (K - 1) + 5 * e) + 2 * e * B * case["G"] * N + 4 * D * (N + K + 3),
                "flops": B * D * (8 * N + 2 * K + 30)}
    T = case["T"]
    if case["op"] == "conv":
        K = case["K"]
        if case["train"]:
            return {"bytes": 4 * e * B * T * D + 4 * D * (K + 1) * 2, "flops": B * T * D * (6 * K + 30)}
        return {"bytes": 2 * e * B * T * D + 8 * B * (K - 1) * D, "flops": B * T * D * (2 * K + 8)}
    N, G = case["N"], case["G"]
    states = 4 * B * D * N * (2 if case["carry"] else 1)
    if case["train"]:
        return {"bytes": e * (8 * B * T * D + 4 * B * T * G * N) + 8 * D * (N + 2) + 2 * states, "flops": B * T * D * (24 * N + 60)}
    return {"bytes": e * (4 * B * T * D + 2 * B * T * G * N) + 4 * D * (N + 2) + states, "flops": B * T * D * (7 * N + 30)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    d = {k: (v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v) for k, v in s.items()}
    return {"scan": _exact_scan, "conv": _exact_conv, "step": _exact_step, "adamw": _exact_adamw}[case["op"]](case, d)


def _exact_scan(case, d):
    """Step by step, and the gradients step by step backwards."""
    B, T, D, N, G = case["B"], case["T"], case["D"], case["N"], case["G"]
    f = torch.nn.functional
    ends = d["lengths"].tolist() if d["lengths"] is not None else [T] * B
    live = torch.tensor([[1.0 if t < n else 0.0 for n in ends] for t in range(T)], dtype=torch.float64, device=DEV)[:, :, None]
    group = torch.arange(D, device=DEV) // (D // G)
    A = d["a"]
    h = d["h0"].clone() if d["h0"] is not None else torch.zeros(B, D, N, dtype=torch.float64, device=DEV)
    kept = torch.empty(T, B, D, N, dtype=torch.float64, device=DEV) if case["train"] else None
    raw = d["dt"] + d["dt_bias"]
    delta = torch.logaddexp(raw, torch.zeros_like(raw)) * live.transpose(0, 1)
    y = torch.empty(B, T, D, dtype=torch.float64, device=DEV)
    for t in range(T):
        if kept is not None:
            kept[t] = h
        h = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * d["x"][:, t])[:, :, None] * d["b"][:, t][:, group]
        y[:, t] = torch.einsum("bdn,bdn->bd", h, d["c"][:, t][:, group]) + d["skip"] * d["x"][:, t]
    live = live.transpose(0, 1)
    out = y * f.silu(d["gate"]) * live
    if not case["train"]:
        return out, h
    dy = d["dy"] * live
    sig = torch.sigmoid(d["gate"])
    got = {"y": out, "state": h, "d_gate": dy * y * (sig + d["gate"] * sig * (1 - sig))}
    g = dy * d["gate"] * sig
    q = d["dh"].clone() if d["dh"] is not None else torch.zeros_like(h)
    d_x, d_raw = torch.empty_like(y), torch.empty_like(y)
    d_a = torch.zeros_like(A)
    d_b, d_c = torch.empty_like(d["b"]), torch.empty_like(d["c"])
    onto = torch.zeros(G, D, dtype=torch.float64, device=DEV)
    onto[group, torch.arange(D, device=DEV)] = 1.0
    for t in reversed(range(T)):
        decay = torch.exp(delta[:, t, :, None] * A)
        bt, ct = d["b"][:, t][:, group], d["c"][:, t][:, group]
        now = decay * kept[t] + (delta[:, t] * d["x"][:, t])[:, :, None] * bt
        q = q + ct * g[:, t, :, None]
        d_c[:, t] = torch.matmul(onto, now * g[:, t, :, None])
        d_b[:, t] = torch.matmul(onto, q * (delta[:, t] * d["x"][:, t])[:, :, None])
        w = q * decay * kept[t]
        d_a += (w * delta[:, t, :, None]).sum(0)
        qb = (q * bt).sum(-1)
        d_x[:, t] = qb * delta[:, t] + g[:, t] * d["skip"]
        d_raw[:, t] = ((w * A).sum(-1) + qb * d["x"][:, t]) * torch.sigmoid(raw[:, t]) * live[:, t]
        q = q * decay
    got |= {"d_x": d_x, "d_dt": d_raw, "d_a": d_a, "d_b": d_b, "d_c": d_c, "d_skip": (g * d["x"]).sum((0, 1)),
            "d_dt_bias": d_raw.sum((0, 1))}
    if d["h0"] is not None:
        got["d_h0"] = q
    return got


def _exact_conv(case, d):
    B, T, D, K = case["B"], case["T"], case["D"], case["K"]
    f = torch.nn.functional
    ends = d["lengths"].tolist() if d["lengths"] is not None else [T] * B
    before = d["h0"] if d["h0"] is not None else torch.zeros(B, K - 1, D, dtype=torch.float64, device=DEV)
    y = torch.zeros(B, T, D, dtype=torch.float64, device=DEV)
    last = torch.empty(B, K - 1, D, dtype=torch.float64, device=DEV)
    d_x, d_h0 = torch.zeros_like(y), torch.zeros_like(last)
    d_w, d_wb = torch.zeros_like(d["w"]), torch.zeros_like(d["wb"])
    for i, n in enumerate(ends):                                          # one sequence after the other, at its own length
        xs = torch.cat([before[i], d["x"][i, :n]], 0)
        last[i] = xs[n:]
        d_xs = torch.zeros_like(xs)
        if n:
            pre = d["wb"] + sum(xs[k:k + n] * d["w"][:, k] for k in range(K))
            y[i, :n] = f.silu(pre)
        if not case["train"]:
            continue
        if d["dh"] is not None:
            d_xs[n:] += d["dh"][i]
        if n:
            sig = torch.sigmoid(pre)
            ds = d["dy"][i, :n] * (sig + pre * sig * (1 - sig))
            for k in range(K):
                d_xs[k:k + n] += ds * d["w"][:, k]
                d_w[:, k] += (ds * xs[k:k + n]).sum(0)
            d_wb += ds.sum(0)
        d_h0[i], d_x[i, :n] = d_xs[:K - 1], d_xs[K - 1:]
    if not case["train"]:
        return y, last
    got = {"y": y, "state": last, "d_x": d_x, "d_w": d_w, "d_wb": d_wb}
    if d["h0"] is not None:
        got["d_h0"] = d_h0
    return got


def _exact_step(case, d):
    f = torch.nn.functional
    D, G = case["D"], case["G"]
    xs = torch.cat([d["conv_state"], d["x"][:, None]], 1)
    x = f.silu(torch.einsum("bkd,dk->bd", xs, d["w"]) + d["wb"])
    seen = x.to(DTYPES[case["dtype"]]).double()                           # (what the first call hands to the second)
    raw = d["dt"] + d["dt_bias"]
    delta = torch.logaddexp(raw, torch.zeros_like(raw))
    group = torch.arange(D, device=DEV) // (D // G)
    h = d["state"] * torch.exp(delta[:, :, None] * d["a"]) + (delta * seen)[:, :, None] * d["b"][:, group]
    y = (torch.einsum("bdn,bdn->bd", h, d["c"][:, group]) + d["skip"] * seen) * f.silu(d["gate"])
    return {"x": x, "y": y, "conv_state": xs[:, 1:], "state": h}


def _exact_adamw(case, d):
    """The first step, from moments of zero: the 8-bit codes are found in their tables of values."""
    got = {"p": [], "m": [], "v": []}
    table_m = (torch.arange(128, dtype=torch.float64, device=DEV) / 127.0) ** 2
    table_v = (torch.arange(256, dtype=torch.float64, device=DEV) / 255.0) ** 4
    for p, g in zip(d["p"], d["g"]):
        p, g = p.double(), g.double()
        m, v = (1.0 - BETA1) * g, (1.0 - BETA2) * g * g
        got["p"].append(p * (1.0 - LR * DECAY) - LR * (m / (1.0 - BETA1)) / (torch.sqrt(v / (1.0 - BETA2)) + EPS))
        if case["bits"] == 8:
            n = g.numel()
            block = torch.arange(n, device=DEV) // BLOCK
            u = torch.remainder(torch.remainder(torch.arange(n, device=DEV) * WEYL_I, 2 ** 32) + WEYL_T, 2 ** 32)
            u = (u.double() + 0.5) / 2.0 ** 32
            count = (n + BLOCK - 1) // BLOCK
            for x, table, name, share in ((m, table_m, "m", u), (v, table_v, "v", 1.0 - u)):
                size = x.reshape(-1).abs()
                top = torch.zeros(count, dtype=torch.float64, device=DEV).scatter_reduce_(0, block, size, "amax")
                top = top.float().double()[block]
                part = torch.where(top > 0, size / top.clamp(min=1e-300), torch.zeros_like(size)).clamp_(max=1.0)
                low = (torch.bucketize(part, table, right=True) - 1).clamp_(max=table.numel() - 2)
                code = low + (part - table[low] > share * (table[low + 1] - table[low])).long()
                if name == "v":
                    code = torch.where((code < 1) & (size > 0) & (top > 0), torch.ones_like(code), code)
                got[name].append((torch.sign(x.reshape(-1)) * top * table[code]).view(g.shape))
        else:
            got["m"].append(m)
            got["v"].append(v)
    return got
