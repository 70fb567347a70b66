"""vsv.ssm on the GPU against its plain 64-bit forms, elementwise: half a step of the output's type, plus K half steps of
float32 at the size of the terms that make it up.

Scan: every step of either recurrence rounds at most 8 times (time step: softplus 4e-9 + 5 roundings, shared; exponent's two
products, the exponential's ulp, the state's product and sum), over at most T steps, and sums over the N states and the
activations add fewer than 64 + 2 N; sums over a sequence, a batch or a group's channels add one per term.  Convolution: K + 1
products and sums, the activation and its slope fewer than 32; sums over time and batch one per term."""
import pytest
import torch

from ssm_reference import SCAN_PLANS, check, conv_ref, scan_ref

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _rand(seed):
    g = torch.Generator().manual_seed(seed)
    return (lambda *s, scale=1.0, dtype=torch.float32: (torch.randn(*s, generator=g) * scale).to(dtype).cuda()), g


def _scan_case(seed, B, T, D, N, G, dtype, parts="sgbh"):
    r, g = _rand(seed)
    t = DT[dtype]
    a = -(torch.arange(1, N + 1) * (1 + 0.2 * torch.rand(D, N, generator=g))).cuda()
    return dict(x=r(B, T, D, dtype=t), dt=r(B, T, D, scale=0.5, dtype=t), a=a, b=r(B, T, G, N, dtype=t), c=r(B, T, G, N, dtype=t),
                skip=r(D) if "s" in parts else None, gate=r(B, T, D, dtype=t) if "g" in parts else None,
                dt_bias=r(D, scale=1.5) - 3.0 if "b" in parts else None, h0=r(B, D, N) if "h" in parts else None,
                dy=r(B, T, D, dtype=t), dh=r(B, D, N))


def _scan_run(s, lengths=None, softplus=True, grads=True):
    from vsv.ssm import ssm_scan
    names = [n for n in ("x", "dt", "a", "b", "c", "skip", "gate", "dt_bias", "h0") if s[n] is not None]
    leaves = {n: s[n].detach().requires_grad_(grads) for n in names}
    get = leaves.get
    y, h = ssm_scan(get("x"), get("dt"), get("a"), get("b"), get("c"), get("skip"), get("gate"), dt_bias=get("dt_bias"),
                    softplus=softplus, initial_state=get("h0"), lengths=lengths, return_state=True)
    got = {"y": y, "state": h}
    if grads:
        got |= dict(zip(names, torch.autograd.grad((y, h), list(leaves.values()), (s["dy"], s["dh"]))))
    return got


def _scan_check(s, got, lengths=None, softplus=True):
    args = [s[n] for n in ("x", "dt", "a", "b", "c", "skip", "gate", "dt_bias", "h0")] + [lengths, softplus]
    grads = len(got) > 2
    want = scan_ref(*args, s["dy"] if grads else None, s["dh"] if grads else None)
    size = scan_ref(*args, s["dy"] if grads else None, s["dh"] if grads else None, absolute=True)
    B, T, D = s["x"].shape
    N, G = s["a"].shape[1], s["b"].shape[2]
    base = 8 * T + 64 + 2 * N
    extra = {"a": B * T, "skip": B * T, "dt_bias": B * T, "b": D // G, "c": D // G}
    for n, v in got.items():
        check(n, v, want[n], size[n], base + extra.get(n, 0))


SHAPES = [(1, 1, 1, 1, 1), (2, 7, 3, 2, 1), (3, 8, 64, 4, 1), (1, 9, 65, 16, 1), (2, 33, 130, 16, 2), (2, 64, 96, 13, 3), (5, 61, 100, 16, 1),
          (1, 130, 257, 8, 1), (1, 515, 70, 5, 1), (64, 3, 36, 16, 1), (1, 1100, 24, 16, 2)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan(shape, dtype):
    s = _scan_case(3, *shape, dtype)
    _scan_check(s, _scan_run(s))


@pytest.mark.parametrize("parts", ["", "s", "g", "b", "h", "gh"])
@pytest.mark.parametrize("softplus", [True, False])
def test_scan_without_some_of_its_parts(parts, softplus):
    if not softplus and "b" in parts:
        pytest.skip("a bias of -3 makes the time steps negative: the states themselves overflow, in 64 bits too")
    s = _scan_case(4, 2, 21, 70, 16, 1, "fp32", parts)
    if not softplus:
        s["dt"] = s["dt"].abs() * 0.1
    _scan_check(s, _scan_run(s, softplus=softplus), softplus=softplus)


def test_scan_time_steps_as_they_are():
    s = _scan_case(13, 2, 45, 70, 16, 1, "fp32")
    s["dt"], s["dt_bias"] = s["dt"].abs() * 0.1, s["dt_bias"].abs() * 0.01
    _scan_check(s, _scan_run(s, softplus=False), softplus=False)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T, lengths", [(1, [0, 1, 0]), (37, [0, 37, 8]), (40, [39, 1, 16]), (300, [300, 17, 129]), (300, [0, 0, 0])])
def test_scan_padded(T, lengths, dtype):
    """Padding holds NaN and infinities: it is never read, its outputs and gradients are zero."""
    s = _scan_case(5, 3, T, 72, 16, 2, dtype)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    pad = torch.arange(T).cuda()[None, :] >= n[:, None]
    for k, v in (("x", float("nan")), ("dt", float("inf")), ("gate", float("nan")), ("dy", float("nan")), ("b", float("inf")), ("c", float("nan"))):
        s[k][pad] = v
    got = _scan_run(s, n)
    _scan_check(s, got, n)
    for k in ("y", "x", "dt", "gate", "b", "c"):
        assert (got[k][pad] == 0).all(), k
    for i, m in enumerate(lengths):
        if m == 0:
            assert torch.equal(got["state"][i], s["h0"][i]) and torch.equal(got["h0"][i], s["dh"][i])
    outside = torch.tensor([m if m < T else T + 1000 for m in lengths]).cuda()           # int64, beyond the end: the end
    again = _scan_run(s, torch.where(outside == 0, outside - 5, outside))
    assert all(torch.equal(got[k], again[k]) for k in got)


def test_scan_one_step_whatever_its_stride():
    """A single step's time stride is of no account, however large."""
    s = _scan_case(14, 3, 1, 65, 16, 1, "fp32")
    want = _scan_run(s)
    v = dict(s)
    for n in ("x", "dt", "gate"):
        v[n] = torch.as_strided(s[n], (3, 1, 65), (65, 2**40, 1))
    got = _scan_run(v)
    assert all(torch.equal(got[k], want[k]) for k in want)
    wide = torch.zeros(1, device="cuda").expand(2, 2**27)                                # two steps of 2^27 channels: refused, not wrapped
    from vsv.ssm import ssm_scan
    with pytest.raises(ValueError, match="channels"):
        ssm_scan(wide.unsqueeze(0), wide.unsqueeze(0), torch.zeros(1, 1, device="cuda").expand(2**27, 1), torch.zeros(1, 2, 1, device="cuda"),
                 torch.zeros(1, 2, 1, device="cuda"))


def test_scan_of_nothing():
    for B, T in ((2, 0), (0, 5), (0, 0)):
        s = _scan_case(6, B, T, 40, 16, 1, "fp32")
        got = _scan_run(s)
        assert got["y"].shape == (B, T, 40)
        assert torch.equal(got["state"], s["h0"]) and torch.equal(got["h0"], s["dh"])
        for k in ("a", "skip", "dt_bias"):
            assert (got[k] == 0).all() and got[k].shape == s[k].shape


def test_scan_extreme_time_steps():
    """Time steps from e^-60 to 80 (softplus's both ends), a state that is forgotten at once, one that never decays."""
    s = _scan_case(7, 2, 40, 64, 16, 1, "fp32")
    s["dt"] = torch.linspace(-60, 80, 40).cuda()[None, :, None].expand(2, 40, 64).contiguous()
    s["dt_bias"] = None
    s["a"][:, 0] = 0.0
    s["a"][:, 1] = -1e4
    got = _scan_run(s, grads=False)
    want = scan_ref(*[s[n] for n in ("x", "dt", "a", "b", "c", "skip", "gate", "dt_bias", "h0")], None)
    size = scan_ref(*[s[n] for n in ("x", "dt", "a", "b", "c", "skip", "gate", "dt_bias", "h0")], None, absolute=True)
    # (an exponent delta a of up to 1280 is rounded twice: the decay is off by 2 |delta a| half steps, but then below e^-|delta a|:
    # |u| e^-|u| <= 1/e.  The bound of the ordinary case holds.)
    for n in ("y", "state"):
        check(n, got[n], want[n], size[n], 8 * 40 + 96)


def _strided(s):
    """The same values as views: x, gate halves of one tensor, dt transposed time, b, c pieces of a projection."""
    B, T, D = s["x"].shape
    G, N = s["b"].shape[2:]
    xz = torch.cat([s["x"], s["gate"]], 2)
    bc = torch.cat([torch.zeros(B, T, 3, device="cuda", dtype=xz.dtype), s["b"].flatten(2), s["c"].flatten(2)], 2)
    v = dict(s)
    v["x"], v["gate"] = xz.chunk(2, 2)
    v["dt"] = s["dt"].transpose(0, 1).contiguous().transpose(0, 1)
    _, b, c = bc.split([3, G * N, G * N], 2)
    v["b"], v["c"] = b.unflatten(2, (G, N)), c.unflatten(2, (G, N))
    v["dy"] = s["dy"].transpose(1, 2).contiguous().transpose(1, 2)                        # last dimension not contiguous
    return v


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N, G", [(16, 1), (7, 2), (3, 1)])
def test_scan_views_equal_copies(N, G, dtype):
    s = _scan_case(8, 3, 50, 66, N, G, dtype)
    v = _strided(s)
    assert not v["x"].is_contiguous() and not v["b"].is_contiguous() and v["dy"].stride(-1) != 1
    got, again = _scan_run(s), _scan_run(v)
    for k in got:
        assert torch.equal(got[k], again[k]), k


def test_scan_broadcast_inputs():
    """Operands expanded over the batch and over time: read through their zero strides, their gradients the sums."""
    s = _scan_case(9, 4, 30, 65, 16, 1, "fp32")
    from vsv.ssm import ssm_scan
    b1, dt1 = s["b"][:1].clone().requires_grad_(True), s["dt"][:, :1].clone().requires_grad_(True)
    y = ssm_scan(s["x"], dt1.expand(4, 30, 65), s["a"], b1.expand(4, 30, 1, 16).squeeze(2), s["c"].squeeze(2), s["skip"], s["gate"])
    gb, gd = torch.autograd.grad(y, (b1, dt1), s["dy"])
    s["b"], s["dt"] = b1.detach().expand(4, 30, 1, 16).contiguous(), dt1.detach().expand(4, 30, 65).contiguous()
    s["dt_bias"] = s["h0"] = None
    s["dh"].zero_()
    got = _scan_run(s)
    assert torch.equal(y.detach(), got["y"].detach())
    assert torch.allclose(gb, got["b"].sum(0, keepdim=True), rtol=1e-6, atol=1e-6)
    assert torch.allclose(gd, got["dt"].sum(1, keepdim=True), rtol=1e-6, atol=1e-5)
    ssm_scan(s["x"].requires_grad_(True), s["dt"], s["a"], s["b"], s["c"]).sum().backward()    # (an expanded gradient)
    assert s["x"].grad.shape == s["x"].shape


def test_scan_gradient_of_the_state_alone_and_of_some_inputs():
    from vsv.ssm import ssm_scan
    s = _scan_case(10, 2, 19, 64, 16, 1, "fp32")
    full = dict(s, dy=torch.zeros_like(s["dy"]))
    want = _scan_run(full)
    x, a = s["x"].clone().requires_grad_(True), s["a"].clone().requires_grad_(True)
    y, h = ssm_scan(x, s["dt"], a, s["b"], s["c"], s["skip"], s["gate"], dt_bias=s["dt_bias"], initial_state=s["h0"], return_state=True)
    gx, ga = torch.autograd.grad(h, (x, a), s["dh"])
    assert torch.equal(gx, want["x"]) and torch.equal(ga, want["a"])
    with pytest.raises(RuntimeError):                                                     # no second derivatives
        y, = (ssm_scan(x, s["dt"], a, s["b"], s["c"]),)
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        g.sum().backward()


def test_scan_is_the_same_every_time_and_in_pieces():
    """Bit-equal from run to run; a prompt in two pieces, the state handed over, to rounding."""
    s = _scan_case(11, 3, 700, 200, 16, 1, "fp32")
    one, two = _scan_run(s), _scan_run(s)
    assert all(torch.equal(one[k], two[k]) for k in one)
    from vsv.ssm import ssm_scan
    h, ys = s["h0"], []
    for lo, hi in ((0, 1), (1, 333), (333, 700)):
        cut = [s[n][:, lo:hi] for n in ("x", "dt", "b", "c", "gate")]
        y, h = ssm_scan(cut[0], cut[1], s["a"], cut[2], cut[3], s["skip"], cut[4], dt_bias=s["dt_bias"], initial_state=h, return_state=True)
        ys.append(y)
    _scan_check(s, {"y": torch.cat(ys, 1), "state": h})


def test_scan_long():
    """4100 steps of few rows (the time axis is split), every gradient, with a padded row."""
    s = _scan_case(12, 2, 4100, 40, 16, 1, "fp32")
    n = torch.tensor([4100, 2049], dtype=torch.int32).cuda()
    _scan_check(s, _scan_run(s, n), n)


def test_offsets_beyond_32_bits():
    """Outputs and inputs past element 2^31."""
    from vsv.ssm import short_conv, ssm_scan
    T, D = 1_050_000, 2048
    x = torch.zeros(1, T, D, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(1, 50, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    x[:, -50:] = tail
    w = torch.randn(D, 4, generator=torch.Generator().manual_seed(2)).cuda()
    y, h = short_conv(x, w, return_state=True)
    y2, h2 = short_conv(tail, w, initial_state=torch.zeros(1, 3, D, device="cuda"), return_state=True)
    assert torch.equal(y[:, -50:], y2) and torch.equal(h, h2) and (y[0, ::4099, 0][:-1] == 0).all()
    del y
    r, _ = _rand(3)
    dt, a, b = r(1, 50, D, dtype=torch.bfloat16), -torch.rand(D, 4).cuda(), r(1, 50, 1, 4, dtype=torch.bfloat16)
    big = torch.as_strided(x, (2, 50, D), (x.numel() - 50 * D, D, 1))                     # row 1: the tail
    y = ssm_scan(big, dt.expand(2, 50, D), a, b.expand(2, 50, 1, 4), b.expand(2, 50, 1, 4))
    assert torch.equal(y[1:], ssm_scan(tail, dt, a, b, b)) and (y[0] == 0).all()
    del x, big
    B = 2**31 // (16 * D) + 3                                                             # y itself past 2^31
    y = ssm_scan(tail[:, :16].expand(B, 16, D), dt[:, :16].expand(B, 16, D), a, b[:, :16].expand(B, 16, 1, 4), b[:, :16].expand(B, 16, 1, 4))
    assert torch.equal(y[-1], y[0]) and y[0].abs().sum() > 0


# ---- convolution -------------------------------------------------------------------------------------------------

def _conv_case(seed, B, T, D, K, dtype):
    r, _ = _rand(seed)
    t = DT[dtype]
    return dict(x=r(B, T, D, dtype=t), w=r(D, K), bias=r(D), h0=r(B, K - 1, D).to(t).float(), dy=r(B, T, D, dtype=t), dh=r(B, K - 1, D))


def _conv_run(s, lengths=None, silu=True):
    from vsv.ssm import short_conv
    names = [n for n in ("x", "w", "bias", "h0") if s[n] is not None]
    leaves = {n: s[n].detach().requires_grad_(True) for n in names}
    y, h = short_conv(leaves["x"], leaves["w"], leaves.get("bias"), silu=silu, initial_state=leaves.get("h0"), lengths=lengths, return_state=True)
    return {"y": y, "state": h, **dict(zip(names, torch.autograd.grad((y, h), list(leaves.values()), (s["dy"], s["dh"]), allow_unused=True)))}


def _conv_check(s, got, lengths=None, silu=True):
    args = [s[n] for n in ("x", "w", "bias", "h0")] + [lengths, silu, s["dy"], s["dh"]]
    want, size = conv_ref(*args), conv_ref(*args, absolute=True)
    B, T, _ = s["x"].shape
    assert torch.equal(got["state"].detach().double().cpu(), want["state"])                    # copies of inputs
    for n, v in got.items():
        if n != "state" and v is not None:
            check(n, v, want[n], size[n], 48 + (B * T if n in ("w", "bias") else 0))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("K", [1, 2, 3, 4])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 2, 8), (3, 33, 40), (2, 100, 515), (1, 515, 128)])
def test_conv(shape, K, dtype):
    s = _conv_case(20, *shape, K, dtype)
    for silu in (True, False):
        _conv_check(s, _conv_run(s, silu=silu), silu=silu)
    s["bias"] = s["h0"] = None
    _conv_check(s, _conv_run(s))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("K", [2, 4])
@pytest.mark.parametrize("T, lengths", [(1, [0, 1, 0]), (40, [0, 40, 2]), (70, [31, 32, 33]), (100, [1, 97, 64])])
def test_conv_padded(T, lengths, K, dtype):
    s = _conv_case(21, 3, T, 48, K, dtype)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    pad = torch.arange(T).cuda()[None, :] >= n[:, None]
    s["x"][pad], s["dy"][pad] = float("nan"), float("inf")
    got = _conv_run(s, n)
    _conv_check(s, got, n)
    assert (got["y"][pad] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_conv_views_equal_copies(dtype):
    s = _conv_case(22, 3, 45, 64, 4, dtype)
    got = _conv_run(s)
    wide = torch.zeros(3, 45, 131, device="cuda", dtype=s["x"].dtype)
    for at in (0, 1, 67):                                                                  # rows on and off 16 bytes
        v = dict(s)
        wide[:, :, at:at + 64] = s["x"]
        v["x"] = wide[:, :, at:at + 64]
        again = _conv_run(v)
        assert all(torch.equal(got[k], again[k]) for k in got), at
    v = dict(s, x=s["x"].transpose(1, 2).contiguous().transpose(1, 2), dy=s["dy"][:, :1].expand(3, 45, 64))
    want = _conv_run(dict(s, dy=s["dy"][:, :1].expand(3, 45, 64).contiguous()))
    again = _conv_run(v)
    assert all(torch.equal(want[k], again[k]) for k in got)


def test_conv_of_nothing():
    for B, T in ((2, 0), (0, 5)):
        s = _conv_case(23, B, T, 24, 4, "fp32")
        got = _conv_run(s)
        assert got["y"].shape == (B, T, 24) and torch.equal(got["state"], s["h0"]) and torch.equal(got["h0"], s["dh"])
        assert (got["w"] == 0).all() and (got["bias"] == 0).all()


# ---- single tokens -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B, D, N, G, K", [(1, 1, 1, 1, 1), (3, 70, 16, 1, 4), (2, 128, 8, 2, 3), (5, 33, 5, 3, 2), (1, 2048, 16, 1, 4), (65, 257, 13, 1, 4)])
def test_steps(B, D, N, G, K, dtype):
    """Three tokens one after the other against the same three as a sequence in 64 bits."""
    from vsv.ssm import short_conv_step, ssm_step
    s, k = _scan_case(30, B, 3, D, N, G, dtype), _conv_case(31, B, 3, D, K, dtype)
    state, conv_state = s["h0"].clone(), k["h0"].clone()
    ver = state._version
    ys, cs = [], []
    for t in range(3):
        cs.append(short_conv_step(k["x"][:, t], conv_state, k["w"], k["bias"]))
        ys.append(ssm_step(s["x"][:, t], s["dt"][:, t], s["a"], s["b"][:, t], s["c"][:, t], s["skip"], s["gate"][:, t], state=state, dt_bias=s["dt_bias"]))
    assert state._version > ver
    _scan_check(s, {"y": torch.stack(ys, 1), "state": state})
    args = [k[n] for n in ("x", "w", "bias", "h0")] + [None, True]
    check("conv", torch.stack(cs, 1), conv_ref(*args)["y"], conv_ref(*args, absolute=True)["y"], 48)
    assert torch.equal(conv_state.double().cpu(), conv_ref(*args)["state"])
    from vsv.ssm import short_conv
    assert torch.equal(short_conv(k["x"], k["w"], k["bias"], initial_state=k["h0"]), torch.stack(cs, 1))    # bit for bit


def test_steps_touch_nothing_else():
    """A state inside a larger buffer: the rows before and behind it stay as they were; no gradient is refused, not dropped."""
    from vsv.ssm import short_conv_step, ssm_step
    s = _scan_case(32, 4, 1, 70, 13, 1, "fp32")
    pool = torch.full((6, 70, 13), 7.0, device="cuda")
    cpool = torch.full((6, 2, 70), 7.0, device="cuda")
    ssm_step(s["x"][:, 0], s["dt"][:, 0], s["a"], s["b"][:, 0], s["c"][:, 0], state=pool[1:5])
    short_conv_step(s["x"][:, 0], cpool[1:5], torch.randn(70, 3, device="cuda"))
    for p in (pool, cpool):
        assert (p[0] == 7).all() and (p[5] == 7).all()
    assert not (pool[1:5] == 7).any()
    assert (cpool[1:5, 0] == 7).all() and torch.equal(cpool[1:5, 1], s["x"][:, 0])       # (moved up by one row, the token behind)
    with pytest.raises(RuntimeError, match="no gradient"):
        ssm_step(s["x"][:, 0], s["dt"][:, 0], s["a"].requires_grad_(True), s["b"][:, 0], s["c"][:, 0], state=pool[1:5])


# ---- as a program uses them --------------------------------------------------------------------------------------

def test_memory_prompt_then_tokens_equals_the_whole():
    """SsmMemory over 40 days, then 8 more day by day, against 48 days at once, with a padded row; to the rounding of the
    float32 projections in between."""
    from vsv.ssm import SsmMemory
    torch.manual_seed(0)
    mem = SsmMemory(28, 100).cuda()
    x = torch.randn(3, 48, 28, device="cuda")
    with torch.no_grad():
        want, (cw, hw) = mem(x)
        y, state = mem(x[:, :40])
        got = [y]
        for t in range(40, 48):
            got.append(mem.step(x[:, t], state).unsqueeze(1))
        n = torch.tensor([48, 5, 0], device="cuda")
        yp, (cp, hp) = mem(x, lengths=n)
    got = torch.cat(got, 1)
    # (two orders of the same float32 sums of 28 to 100 products each, three layers deep: 100 half steps a layer at most)
    tol = 300 * 2.0 ** -24
    assert (got - want).abs().max() <= tol * want.abs().max() * 10
    assert (state[1] - hw).abs().max() <= tol * hw.abs().max() * 10 and (state[0] - cw).abs().max() <= tol * cw.abs().max() * 10
    assert torch.allclose(yp[0], want[0], rtol=0, atol=(tol * want.abs().max() * 10).item()) and (yp[1, 5:] == 0).all() and (yp[2] == 0).all()
    assert (hp[2] == 0).all() and (cp[2] == 0).all()


def test_memory_training_step():
    """Forward, loss, backward, optimizer step with 8-bit moments, two steps: every parameter gets the gradient that the plain
    form gives, and moves."""
    from vsv.optim import AdamW
    from vsv.ssm import SsmMemory
    torch.manual_seed(1)
    mem = SsmMemory(12, 36, state_size=8, taps=3).cuda()
    opt = AdamW(mem.parameters(), lr=1e-3, state_bits=8)
    x, target = torch.randn(4, 30, 12, device="cuda"), torch.randn(4, 30, 36, device="cuda")
    for _ in range(2):
        opt.zero_grad()
        y, _ = mem(x)
        ((y - target) ** 2).mean().backward()
        ref = _memory_gradients(mem, x, target)
        for n, p in mem.named_parameters():
            # (float32 projections between the operators: 30 x 4 x 36 terms in a sum, 64 roundings around each)
            tol = (30 * 4 + 36 + 64 + 8 * 30) * 2.0 ** -24 * 40
            assert (p.grad.double().cpu() - ref[n]).abs().max() <= tol * (ref[n].abs().max() + 1e-3), n
        before = [p.detach().clone() for p in mem.parameters()]
        opt.step()
        assert all(not torch.equal(b, p) for b, p in zip(before, mem.parameters()))


def _memory_gradients(mem, x, target):
    """The same memory written with elementary operations in 64 bits on the CPU, differentiated by autograd."""
    P = {n: p.detach().double().cpu().requires_grad_(True) for n, p in mem.named_parameters()}
    x, target = x.double().cpu(), target.double().cpu()
    f = torch.nn.functional
    u, gate = (x @ P["in_proj.weight"].t() + P["in_proj.bias"]).chunk(2, -1)
    K, n, r = mem.taps, mem.state_size, mem.dt_rank
    up = torch.cat([torch.zeros(x.shape[0], K - 1, u.shape[2]).double(), u], 1)
    u = f.silu(sum(up[:, k:k + x.shape[1]] * P["conv_weight"][:, k] for k in range(K)) + P["conv_bias"])
    dt, b, c = (u @ P["x_proj.weight"].t()).split([r, n, n], -1)
    delta = f.softplus(dt @ P["dt_proj.weight"].t() + P["dt_bias"], threshold=100)
    A = -torch.exp(P["a_log"])
    h, ys = torch.zeros(x.shape[0], u.shape[2], n).double(), []
    for t in range(x.shape[1]):
        h = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * u[:, t])[:, :, None] * b[:, t, None]
        ys.append(((h * c[:, t, None]).sum(-1) + P["skip"] * u[:, t]) * f.silu(gate[:, t]))
    loss = ((torch.stack(ys, 1) - target) ** 2).mean()
    return dict(zip(P, torch.autograd.grad(loss, list(P.values()))))


def test_captured_and_replayed():
    """Forward and backward in one HIP graph, replayed on new inputs between eager work; two graphs alive at once."""
    r, _ = _rand(40)
    graphs = []
    for T in (90, 517):
        s = _scan_case(41, 2, T, 72, 16, 1, "fp32")
        k = _conv_case(42, 2, T, 72, 4, "fp32")
        _scan_run(s); _conv_run(k)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side, capture_error_mode="thread_local"):
                out = _scan_run(s), _conv_run(k)
        graphs.append((g, s, k, out))
    for turn in range(3):
        for g, s, k, _ in graphs:
            for t in (s["x"], s["dt"], s["dy"], s["a"], k["x"], k["dy"]):
                t.copy_(-torch.rand_like(t) if t is s["a"] else torch.randn_like(t))
            torch.cuda.synchronize()
            g.replay()
        torch.cuda.synchronize()
        for g, s, k, (so, ko) in graphs:
            for got, want in ((so, _scan_run(s)), (ko, _conv_run(k))):
                for n in want:
                    assert torch.equal(got[n], want[n]), (turn, n)


def test_on_another_stream():
    s = _scan_case(43, 2, 600, 130, 16, 1, "bf16")
    want = _scan_run(s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _scan_run(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_views_with_their_sign_put_off():
    from vsv.ssm import short_conv, ssm_scan
    z = torch.randn(2, 20, 70, dtype=torch.complex64, device="cuda").conj()
    w = torch.randn(70, 4, dtype=torch.complex64, device="cuda").conj()
    assert z.imag.is_neg() and w.imag.is_neg()
    assert torch.equal(short_conv(z.imag, w.imag), short_conv(z.imag.clone(), w.imag.clone()))
    x, a, b = z.imag, -torch.rand(70, 8, device="cuda"), torch.randn(2, 20, 8, device="cuda")
    assert torch.equal(ssm_scan(x, x, a, b, b, w.imag[:, 0], x), ssm_scan(x.clone(), x.clone(), a, b, b, w.imag[:, 0].clone(), x.clone()))


def test_states_made_in_inference_mode():
    from vsv.ssm import SsmMemory
    mem = SsmMemory(6, 70).cuda()
    x = torch.randn(3, 9, 6, device="cuda")
    with torch.inference_mode():
        whole, _ = mem(x)
        _, state = mem(x[:, :8])
        last = mem.step(x[:, 8], state)
        # (three products of up to 70 terms one after the other, in float32, summed in another order: 3 * 70 * 2^-24 = 1.3e-5 of the
        # terms' sizes, which are up to some times the sums')
        assert (last - whole[:, 8]).abs().max() <= 1e-4 * whole.abs().max()
    kept = [t.clone() for t in state]
    with pytest.raises(RuntimeError, match="[Ii]nference"):                  # torch's own rule, and nothing has been written
        mem.step(x[:, 8], state)
    torch.cuda.synchronize()
    assert all(torch.equal(t, k) for t, k in zip(state, kept))


@pytest.mark.parametrize("T, N, lengths", [(600, 16, [600, 17, 0]), (600, 8, [8, 591, 592]), (47, 16, [47, 40, 3]), (100, 4, [100, 41, 0]),
                                           (2100, 3, [2100, 2097, 1000]), (127, 5, [127, 120, 9])])
def test_scan_padded_in_many_segments(T, N, lengths):
    """Lengths that end in the first, a middle, the last or in front of every segment."""
    s = _scan_case(44, 3, T, 70, N, 1, "fp32")
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    s["x"][torch.arange(T).cuda()[None, :] >= n[:, None]] = float("nan")
    _scan_check(s, _scan_run(s, n), n)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N", [4, 8, 16])
def test_step_with_b_and_c_anywhere(N, dtype):
    """b and c as pieces of a projection whose rows start on any element."""
    from vsv.ssm import ssm_step
    s = _scan_case(45, 5, 1, 70, N, 2, dtype)
    x, dt, gate, b, c = (s[k][:, 0] for k in ("x", "dt", "gate", "b", "c"))
    states, ys = [], []
    for at, end in ((0, 0), (1, 0), (3, 2), (4, 4)):
        row = torch.cat([torch.full((5, at), 7.0, device="cuda", dtype=b.dtype), b.flatten(1), c.flatten(1),
                         torch.full((5, end), 7.0, device="cuda", dtype=b.dtype)], 1)
        _, vb, vc, _ = row.split([at, 2 * N, 2 * N, end], 1)
        states.append(s["h0"].clone())
        ys.append(ssm_step(x, dt, s["a"], vb.unflatten(1, (2, N)), vc.unflatten(1, (2, N)), s["skip"], gate, state=states[-1], dt_bias=s["dt_bias"]))
    for y, st in zip(ys, states):
        _scan_check(s, {"y": y[:, None], "state": st})
        assert torch.equal(y, ys[0]) and torch.equal(st, states[0])


def test_gradients_past_32_bits():
    """More than 2^31 elements: two sequences of the same inputs have the same outputs and gradients, wherever they lie."""
    from vsv.ssm import short_conv, ssm_scan, ssm_step
    T, D, N = (1 << 20) + 5, 1100, 8
    r = lambda *shape: torch.randn(*shape, device="cuda").to(torch.bfloat16)
    x, b, w = r(1, T, D).expand(2, T, D), r(1, T, N).expand(2, T, N), torch.randn(D, 4, device="cuda")
    a, dy = -torch.rand(D, N, device="cuda") - 0.1, r(1, T, D).expand(2, T, D)
    for call in (lambda t: short_conv(t, w), lambda t: ssm_scan(t, x[:, :t.shape[1]], a, b[:, :t.shape[1]], b[:, :t.shape[1]], gate=x[:, :t.shape[1]])):
        leaf = x.detach().requires_grad_(True)
        y = call(leaf)
        assert y.numel() > 2**31 and torch.equal(y[0], y[1]) and y[1, -1].abs().sum() > 0
        g, = torch.autograd.grad(y, leaf, dy)
        assert torch.equal(g[0], g[1]) and g[1, -1].abs().sum() > 0
        short = call(x[:, :300])                                              # (the front, computed in another number of segments)
        assert (short[1] - y[1, :300]).abs().max() <= 2.0 ** -7 * y[1, :300].abs().max()
        del y, g, leaf, short
    B, D = 33000, 4096
    state = torch.zeros(B, D, 16, device="cuda")
    assert state.numel() > 2**31
    x, b, a = r(1, D).expand(B, D), r(1, 16).expand(B, 16), -torch.rand(D, 16, device="cuda")
    y = ssm_step(x, x, a, b, b, state=state)
    assert torch.equal(y[-1], y[0]) and torch.equal(state[-1], state[0]) and state[-1].abs().sum() > 0


def test_tokens_captured_and_replayed():
    """One token's two steps in a HIP graph: every replay takes the next token and moves the states on, as eager calls do."""
    from vsv.ssm import short_conv_step, ssm_step
    s, k = _scan_case(46, 3, 6, 72, 16, 1, "bf16"), _conv_case(47, 3, 6, 72, 4, "bf16")

    def token(x, dt, b, c, gate, conv_state, state):
        u = short_conv_step(x, conv_state, k["w"], k["bias"])
        return ssm_step(u, dt, s["a"], b, c, s["skip"], gate, state=state, dt_bias=s["dt_bias"])
    inputs = [[t[:, i].clone() for t in (k["x"], s["dt"], s["b"], s["c"], s["gate"])] for i in range(6)]
    want_states = [k["h0"].clone(), s["h0"].clone()]
    want = [token(*i, *want_states) for i in inputs]
    held, states = [t.clone() for t in inputs[0]], [k["h0"].clone(), s["h0"].clone()]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            out = token(*held, *states)
    for i, y in zip(inputs, want):
        for h, t in zip(held, i):
            h.copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)
        (out.float() @ out.float().t()).sum().item()                          # (eager work in between)
    assert all(torch.equal(g, w) for g, w in zip(states, want_states))


def test_two_threads_at_once():
    """Calls of two threads on their own streams, forward and backward, give what each gives alone."""
    import threading
    cases = [_scan_case(48, 2, 300, 130, 16, 1, "fp32"), _scan_case(49, 3, 90, 100, 8, 1, "bf16")]
    want = [_scan_run(s) for s in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = _scan_run(cases[i])
                torch.cuda.current_stream().synchronize()
                wrong.extend(n for n in got if not torch.equal(got[n], want[i][n]))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_forward_mode_is_refused():
    """Forward, in either mode, and backward from an output's gradient that carries a tangent; without one, a dual level changes nothing."""
    import torch.autograd.forward_ad as fwd
    from vsv.ssm import short_conv, ssm_scan
    s, k = _scan_case(50, 2, 9, 8, 4, 1, "fp32"), _conv_case(51, 2, 9, 8, 4, "fp32")
    calls = (lambda x: ssm_scan(x, s["dt"], s["a"], s["b"], s["c"]), lambda x: short_conv(x, k["w"]))
    with fwd.dual_level():
        for call in calls:
            want = call(s["x"])
            for on in (True, False):
                with torch.set_grad_enabled(on), pytest.raises(RuntimeError, match="forward-mode"):
                    call(fwd.make_dual(s["x"], torch.ones_like(s["x"])))
            leaf = s["x"].clone().requires_grad_(True)
            y = call(leaf)
            assert torch.equal(y, want)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, fwd.make_dual(s["dy"], torch.ones_like(s["dy"])), retain_graph=True)
            torch.autograd.grad(y, leaf, s["dy"])


def test_gradients_with_their_sign_put_off():
    """The outputs' and the states' gradients as contiguous negative views."""
    s, k = _scan_case(52, 2, 20, 70, 8, 1, "fp32"), _conv_case(53, 2, 20, 70, 4, "fp32")
    for run, c in ((_scan_run, s), (_conv_run, k)):
        v = dict(c, dy=torch._neg_view(c["dy"]), dh=torch._neg_view(c["dh"]))
        want = run(dict(c, dy=-c["dy"], dh=-c["dh"]))
        assert v["dh"].is_contiguous() and v["dh"].is_neg()
        got = run(v)
        assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("T, N", [(64, 4), (2048, 4), (100, 16), (1100, 16), (300, 8)])
def test_scan_states_that_grow(T, N):
    """Decays whose product over a segment of time leaves float32, over states (backwards: gradients) that are zero there: inputs in
    the last three steps only, the outputs' gradients in the first three."""
    s = _scan_case(54, 2, T, 5, N, 1, "fp32", "s")
    s["a"] = torch.full_like(s["a"], 8.0)                                    # (two tiles of steps of 1: e^128)
    s["dt"] = torch.ones_like(s["dt"])
    s["x"][:, :-3] = 0.0
    s["dy"][:, 3:] = 0.0
    s["dh"].zero_()
    _scan_check(s, _scan_run(s, softplus=False), softplus=False)


@pytest.mark.parametrize("T", [64, 2048])
def test_scan_small_states_that_grow(T):
    """A state of 1e-30 and a state's gradient of the same size, past 1e43 times that in one segment of time, no further."""
    for first in (True, False):
        s = _scan_case(55, 2, T, 5, 4, 1, "fp32", "sh")
        s["a"] = torch.full_like(s["a"], 100.0 / 16.0)
        s["dt"] = torch.zeros_like(s["dt"])
        s["dt"][:, :16 if first else T] = 1.0
        if not first:
            s["dt"][:, :T - 16] = 0.0
        s["x"].zero_()
        s["dy"].zero_()
        s["h0"] *= 1e-30 if first else 0.0
        s["dh"] *= 0.0 if first else 1e-30
        # (the exponent 16 x 6.25 log2 e = 144 is rounded three times: 3 x 100 half steps, within the 8 T + 64 of the bound)
        _scan_check(s, _scan_run(s, softplus=False), softplus=False)


@pytest.mark.parametrize("a", [float("-inf"), -3e38])
@pytest.mark.parametrize("T, N", [(5, 4), (5, 16), (100, 16), (300, 3), (2100, 4)])
def test_scan_states_that_are_forgotten_at_once(T, N, a):
    """a = -inf, and an a whose exponent leaves float32: padding, behind a length or in a last tile, leaves the state alone.  The values
    and gradients are those of a = -1e30, whose decays are 0 too (as an infinity the formula's gradient would be 0 times it)."""
    s = _scan_case(56, 3, T, 6, N, 1, "fp32", "sgh")
    n = torch.tensor([T, T // 2, 0], dtype=torch.int32).cuda()
    s["a"][:, 0] = a
    got = _scan_run(s, n)
    s["a"][:, 0] = -1e30
    _scan_check(s, got, n)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_memory_whatever_its_padding_holds(kind):
    """Outputs, states and every gradient as with zeros there; lengths outside [0, T] count as the nearest of the two."""
    from vsv.ssm import SsmMemory
    torch.manual_seed(3)
    mem = SsmMemory(6, 20).cuda()
    x, dy = torch.randn(4, 11, 6, device="cuda"), torch.randn(4, 11, 20, device="cuda")
    n = torch.tensor([11, 4, 0, 900], dtype=kind, device="cuda")
    pad = torch.arange(11, device="cuda") >= n[:, None]
    got = []
    for fill in (0.0, float("nan"), float("inf")):
        mem.zero_grad()
        leaf = x.clone()
        leaf[pad] = fill
        leaf.requires_grad_(True)
        y, state = mem(leaf, lengths=n)
        (y * dy).sum().backward()
        got.append([y.detach(), *(t.detach() for t in state), leaf.grad, *(p.grad.clone() for p in mem.parameters())])
    assert all(torch.isfinite(t).all() for t in got[0]) and (got[0][3][pad] == 0).all()
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    with pytest.raises(ValueError, match="lengths"):
        mem(x, lengths=[11, 4, 0, 11])
    with pytest.raises(ValueError, match="tensors are on"):
        mem(x, lengths=n.cpu())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", list(SCAN_PLANS), ids=lambda s: SCAN_PLANS[s].replace(" ", "-") + "-" + "x".join(map(str, s)))
def test_scan_however_it_is_divided(shape, dtype):
    """Every kernel that a forward pass can take, elementwise, with lengths, a carried state and every gradient."""
    s = _scan_case(57, *shape, dtype)
    B, T = shape[:2]
    n = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(58), dtype=torch.int32)
    n[0], n[1], n[2] = T, 0, T - 1
    n = n.cuda()
    s["x"][torch.arange(T).cuda()[None, :] >= n[:, None]] = float("nan")
    _scan_check(s, _scan_run(s, n), n)


@pytest.mark.parametrize("B, T, D, dtype", [(64, 1000, 1024, "bf16"), (64, 2100, 1024, "fp16"), (64, 1000, 1024, "fp32"), (64, 500, 515, "fp32"),
                                            (64, 1010, 515, "bf16")])
def test_conv_in_long_chunks(B, T, D, dtype):
    """Chunks of 32 and 64 rows forward, 128 backward (threads: 524288 and 131072 at least, of four channels each or of one): 40 channels, the
    first and the last among them, elementwise with their gradients; lengths that end anywhere in a chunk."""
    s = _conv_case(59, B, T, D, 4, dtype)
    g = torch.Generator().manual_seed(60)
    n = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    n[:4] = torch.tensor([T, T - 1, 64, 127], dtype=torch.int32)
    n = n.cuda()
    got = _conv_run(s, n)
    at = torch.cat([torch.tensor([0, D - 1]), torch.randperm(D, generator=g)[:38]]).cuda()
    part = {k: v[:, :, at] if k in ("x", "h0", "dy", "dh") else v[at] for k, v in s.items()}
    _conv_check(part, {k: v[at] if k in ("w", "bias") else v[:, :, at] for k, v in got.items()}, n)
