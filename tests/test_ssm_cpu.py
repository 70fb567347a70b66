"""vsv.ssm and vsv.optim without a GPU: the references' gradients against differences, and every refusal."""
import ctypes as C

import pytest
import torch

from ssm_reference import SCAN_PLANS, conv_ref, scan_plan, scan_ref


def _case(seed, B=2, T=5, D=4, N=3, G=2, K=3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)        # noqa: E731
    scan = dict(x=r(B, T, D), dt=r(B, T, D), a=-torch.rand(D, N, generator=g, dtype=torch.float64) - 0.2, b=r(B, T, G, N), c=r(B, T, G, N),
                skip=r(D), gate=r(B, T, D), dt_bias=r(D), h0=r(B, D, N))
    conv = dict(x=r(B, T, D), w=r(D, K), bias=r(D), h0=r(B, K - 1, D))
    return scan, conv, r(B, T, D), r(B, D, N), r(B, K - 1, D)


@pytest.mark.parametrize("lengths", [None, [5, 0], [3, 1]])
@pytest.mark.parametrize("flag", [True, False])
def test_reference_gradients_are_the_differences(lengths, flag):
    """Each formula's gradient along a random direction against a central difference of the plain forward: the difference's
    own error is h^2 / 6 of a third derivative, 1e-10 at h = 1e-5, and rounding 1e-16 / h = 1e-11, of values around 10."""
    scan, conv, dy, dh, dc = _case(1)
    h = 1e-5
    loss = lambda o, d: (o["y"] * dy).sum() + (o["state"] * d).sum()        # noqa: E731
    for args, ref, d in ((scan, scan_ref, dh), (conv, conv_ref, dc)):
        got = ref(*args.values(), lengths, flag, dy, d)
        for name, t in args.items():
            v = torch.randn(t.shape, generator=torch.Generator().manual_seed(7), dtype=torch.float64)
            plus = loss(ref(*{**args, name: t + h * v}.values(), lengths, flag), d)
            minus = loss(ref(*{**args, name: t - h * v}.values(), lengths, flag), d)
            slope = ((plus - minus) / (2 * h)).item()
            assert abs(slope - (got[name] * v).sum().item()) <= 1e-7 * (1 + abs(slope)), name


def _scan_tensors(B=2, T=4, D=6, N=4, G=1, dtype=torch.float32):
    z = torch.zeros
    return dict(x=z(B, T, D, dtype=dtype), dt=z(B, T, D, dtype=dtype), a=z(D, N), b=z(B, T, G, N, dtype=dtype), c=z(B, T, G, N, dtype=dtype))


@pytest.mark.parametrize("change, word", [
    (dict(x=torch.zeros(4, 6)), "x must be"),
    (dict(x=torch.zeros(2, 4, 6, dtype=torch.float64)), "x must be"),
    (dict(dt=torch.zeros(2, 4, 6, dtype=torch.bfloat16)), "dt must be"),
    (dict(dt=torch.zeros(2, 5, 6)), "dt must be"),
    (dict(a=torch.zeros(6, 17)), "a must be"),
    (dict(a=torch.zeros(6, 0)), "a must be"),
    (dict(a=torch.zeros(5, 4)), "a must be"),
    (dict(a=torch.zeros(6, 4, dtype=torch.bfloat16)), "a must be"),
    (dict(b=torch.zeros(2, 4, 4, 4)), "b must be"),
    (dict(b=torch.zeros(2, 4, 2, 4)), "groups"),
    (dict(c=torch.zeros(2, 4, 1, 5)), "c must be"),
    (dict(skip=torch.zeros(5)), "skip must be"),
    (dict(gate=torch.zeros(2, 4, 5)), "gate must be"),
    (dict(dt_bias=torch.zeros(6, dtype=torch.float64)), "dt_bias must be"),
    (dict(initial_state=torch.zeros(2, 6, 3)), "initial_state must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths must be"),
    (dict(lengths=torch.zeros(2)), "lengths must be"),
    (dict(lengths=[1, 2]), "lengths must be"),
])
def test_scan_refuses(change, word):
    from vsv.ssm import ssm_scan
    with pytest.raises(ValueError, match=word):
        ssm_scan(**{**_scan_tensors(), **change})


@pytest.mark.parametrize("change, word", [
    (dict(x=torch.zeros(2, 4)), "x must be"),
    (dict(x=torch.zeros(2, 4, 6, dtype=torch.int32)), "x must be"),
    (dict(weight=torch.zeros(6, 5)), "weight must be"),
    (dict(weight=torch.zeros(5, 4)), "weight must be"),
    (dict(weight=torch.zeros(6, 4, dtype=torch.float16)), "weight must be"),
    (dict(bias=torch.zeros(5)), "bias must be"),
    (dict(initial_state=torch.zeros(2, 4, 6)), "initial_state must be"),
])
def test_conv_refuses(change, word):
    from vsv.ssm import short_conv
    with pytest.raises(ValueError, match=word):
        short_conv(**{**dict(x=torch.zeros(2, 4, 6), weight=torch.zeros(6, 4)), **change})


def test_steps_refuse():
    from vsv.ssm import short_conv_step, ssm_step
    x, w = torch.zeros(3, 6), torch.zeros(6, 4)
    a, b = torch.zeros(6, 4), torch.zeros(3, 4)
    for state in (torch.zeros(3, 3, 6, dtype=torch.float64), torch.zeros(3, 4, 6), torch.zeros(3, 6, 3).transpose(1, 2),
                  torch.zeros(1, 3, 6).expand(3, 3, 6)):
        with pytest.raises(ValueError, match="state must be"):
            short_conv_step(x, state, w)
    for state in (None, torch.zeros(3, 4, 6), torch.zeros(1, 6, 4).expand(3, 6, 4), torch.zeros(3, 6, 8)[:, :, ::2]):
        with pytest.raises(ValueError, match="state must be"):
            ssm_step(x, x, a, b, b, state=state)
    with pytest.raises(ValueError, match="b must be"):
        ssm_step(x, x, a, torch.zeros(2, 4), b, state=torch.zeros(3, 6, 4))


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    """An input with a tangent, whether or not gradients are enabled: the output would have none."""
    import torch.autograd.forward_ad as fwd
    from vsv.ssm import short_conv, short_conv_step, ssm_scan, ssm_step
    t = {**_scan_tensors(), "skip": torch.zeros(6), "gate": torch.zeros(2, 4, 6), "dt_bias": torch.zeros(6), "initial_state": torch.zeros(2, 6, 4)}
    conv = dict(x=torch.zeros(2, 4, 6), weight=torch.zeros(6, 3), bias=torch.zeros(6), initial_state=torch.zeros(2, 2, 6))
    step = {k: v[:, 0] if k in ("x", "dt", "b", "c", "gate") else v for k, v in t.items()}
    step["state"] = step.pop("initial_state")
    conv_step = dict(x=torch.zeros(2, 6), state=torch.zeros(2, 2, 6), weight=torch.zeros(6, 3), bias=torch.zeros(6))
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        for call, args in ((ssm_scan, t), (short_conv, conv), (ssm_step, step), (short_conv_step, conv_step)):
            for name, v in args.items():
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(**{**args, name: fwd.make_dual(v, torch.ones_like(v))})
            with pytest.raises(RuntimeError, match="GPU"):                  # (none: the next refusal)
                call(**args)


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
@pytest.mark.parametrize("grad", [True, False])
def test_tracing_is_refused(grad):
    """A trace would hold the outputs of the inputs it was made with."""
    from vsv.ssm import short_conv, short_conv_step, ssm_scan, ssm_step
    t = _scan_tensors()
    b = t["b"]
    with torch.set_grad_enabled(grad):
        for call, x in ((lambda x: ssm_scan(x, x, t["a"], b, b), t["x"]), (lambda x: short_conv(x, torch.zeros(6, 3)), t["x"]),
                        (lambda x: ssm_step(x, x, t["a"], b[:, 0], b[:, 0], state=torch.zeros(2, 6, 4)), t["x"][:, 0]),
                        (lambda x: short_conv_step(x, torch.zeros(2, 2, 6), torch.zeros(6, 3)), t["x"][:, 0])):
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(call, x)


def test_no_cpu_fallback():
    from vsv.optim import AdamW
    from vsv.ssm import short_conv, short_conv_step, ssm_scan, ssm_step
    t = _scan_tensors()
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    for call in (lambda: ssm_scan(**t), lambda: short_conv(t["x"], torch.zeros(6, 2)),
                 lambda: short_conv_step(torch.zeros(2, 6), torch.zeros(2, 1, 6), torch.zeros(6, 2)),
                 lambda: ssm_step(t["x"][:, 0], t["dt"][:, 0], t["a"], t["b"][:, 0], t["c"][:, 0], state=torch.zeros(2, 6, 4)),
                 lambda: AdamW([p]).step()):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_optimizer_refuses():
    from vsv.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4, 3))
    for bad in (dict(state_bits=4), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    for q in (torch.zeros(4, dtype=torch.float64), torch.zeros(4, 3).t()):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(q)])
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, dtype=torch.float64))]})
    assert len(opt.param_groups) == 1
    p.grad = torch.zeros(4, 3).to_sparse()
    with pytest.raises(ValueError, match="gradient"):
        opt.step()
    with pytest.raises(ValueError, match="same number of bits"):
        AdamW([{"params": [p], "state_bits": 8}])
    from vsv.ssm import SsmMemory
    for bad in (dict(state_size=17), dict(state_size=0), dict(taps=5)):
        with pytest.raises(ValueError, match="are built"):
            SsmMemory(4, 8, **bad)
    with pytest.raises(ValueError, match="8 bits"):
        AdamW([p], state_bits=8).load_state_dict({"state": {0: {"step": 1, "exp_avg": torch.zeros(4, 3)}}, "param_groups": opt.state_dict()["param_groups"]})


def test_optimizer_refuses_negative_views():
    """Contiguous tensors whose memory holds the values' opposites: read raw, a step would go the wrong way."""
    from vsv.optim import AdamW
    neg = torch._neg_view(torch.ones(4))
    assert neg.is_contiguous() and neg.is_neg()
    with pytest.raises(ValueError, match="negative"):
        AdamW([torch.nn.Parameter(neg)])
    p = torch.nn.Parameter(torch.ones(4))
    opt = AdamW([p])
    p.data, p.grad = neg, torch.ones(4)
    with pytest.raises(ValueError, match="negative"):
        opt.step()
    p.data = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU"):
        opt.step()
    opt.state[p]["exp_avg"] = torch._neg_view(torch.zeros(4))
    with pytest.raises(ValueError, match="state was made"):
        opt.step()


def test_optimizer_refuses_parameters_that_share_memory():
    from vsv.optim import AdamW
    flat = torch.zeros(24)
    p, q, r = (torch.nn.Parameter(flat[k:k + 8]) for k in (0, 8, 15))
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="twice"):
        AdamW([p, q, p])
    for x in (p, q, r):
        x.grad = torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU"):                          # side by side is fine
        AdamW([p, q]).step()
    with pytest.raises(ValueError, match="share memory"):
        AdamW([p, q, r]).step()
    tied = torch.nn.Parameter(torch.zeros(8))
    opt = AdamW([{"params": [p]}, {"params": [tied]}])
    tied.data, tied.grad = p.data, torch.ones(8)
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    opt = AdamW([{"params": [p]}, {"params": [q]}])
    opt.param_groups[1]["lr"] = -1.0                                         # (a later group's, found before the first is stepped)
    with pytest.raises(ValueError, match="hyper-parameters"):
        opt.step()
    assert opt.state[p]["step"] == 0


def test_optimizer_refuses_other_rules_options():
    from vsv.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(maximize=True), dict(amsgrad=True), dict(decoupled_weight_decay=False)):
        with pytest.raises(ValueError, match="not built"):
            AdamW([{"params": [p], **bad}])
        theirs = torch.optim.AdamW([p]).state_dict()
        theirs["param_groups"][0].update(bad)
        with pytest.raises(ValueError, match="not built"):
            AdamW([p]).load_state_dict(theirs)
    opt = AdamW([p])
    opt.load_state_dict(torch.optim.AdamW([p], lr=0.25).state_dict())          # torch's own, of the same rule
    assert opt.param_groups[0]["lr"] == 0.25


def _stepped(make, sizes=(4, 9, 300), steps=3):
    """Parameters of their own and torch's optimizer after some steps of theirs."""
    g = torch.Generator().manual_seed(5)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g)) for n in sizes]
    opt = make(ps)
    for _ in range(steps):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g)
        opt.step()
    return ps, opt


def test_state_of_a_stepped_torch_optimizer(monkeypatch):
    """Its step counts are tensors: they become numbers, so that the parameters stay together in one call."""
    from vsv import native
    from vsv.optim import AdamW
    ps, theirs = _stepped(lambda q: torch.optim.AdamW(q, lr=1e-2))
    opt = AdamW(ps)
    opt.load_state_dict(theirs.state_dict())
    assert [type(opt.state[p]["step"]) for p in ps] == [int] * 3 and [opt.state[p]["step"] for p in ps] == [3] * 3
    assert all(torch.equal(opt.state[p][k], theirs.state[p][k]) and opt.state[p][k].data_ptr() != theirs.state[p][k].data_ptr()
               for p in ps for k in ("exp_avg", "exp_avg_sq"))
    made = []

    class Native:
        def adamw_step(self, bits, calls):
            made.extend((len(c[0]), c[-1]) for c in calls)
    monkeypatch.setattr(native, "load", Native)
    opt.step()
    assert made == [(3, 4)] and [opt.state[p]["step"] for p in ps] == [4] * 3


def test_hooks_of_load_state_dict():
    """A pre-hook's dictionary is the one that is taken (and checked), a post-hook sees the state as it will be, and its changes stay."""
    from vsv.optim import AdamW
    ps, theirs = _stepped(lambda q: torch.optim.AdamW(q, lr=1e-2))
    ps[0].data = ps[0].data.bfloat16()                                      # (its moments stay float32)
    opt = AdamW(ps)
    seen = []

    def double(_, d):
        return {**d, "state": {i: {**st, "exp_avg": 2 * st["exp_avg"]} for i, st in d["state"].items()}}

    def after(o):
        seen.extend((o.state[p]["step"], o.state[p]["exp_avg"].dtype) for p in ps)
        o.state[ps[1]]["exp_avg"].zero_()
    handles = [opt.register_load_state_dict_pre_hook(double), opt.register_load_state_dict_post_hook(after)]
    saved = theirs.state_dict()
    opt.load_state_dict(saved)
    assert seen == [(3, torch.float32)] * 3
    assert all(torch.equal(opt.state[p]["exp_avg"], k * theirs.state[p]["exp_avg"]) for p, k in zip(ps, (2, 0, 2)))
    assert all(torch.equal(opt.state[p]["exp_avg_sq"], theirs.state[p]["exp_avg_sq"]) for p in ps)
    for h in handles:
        h.remove()
    opt.load_state_dict(saved)                                              # (nothing of the first call is left)
    assert torch.equal(opt.state[ps[1]]["exp_avg"], theirs.state[ps[1]]["exp_avg"])
    opt.register_load_state_dict_pre_hook(lambda _, d: {**d, "state": {0: {**d["state"][0], "exp_avg": torch.zeros(5)}}})
    with pytest.raises(ValueError, match="exp_avg"):
        opt.load_state_dict(saved)


def test_scan_sizes_reach_every_plan():
    """The sizes that the GPU tests take run the kernels they name: the plan written again agrees with the workspace that the
    library asks for (B S (padded states + 1) D floats of a scan in S > 1 segments), and each of the ways is there."""
    from vsv import lib as vlib
    L = vlib.load()
    seen = set()
    for (B, T, D, N, G), what in SCAN_PLANS.items():
        P, S, joined = scan_plan(B, T, D, N, G)
        assert what == ("shared" if P > 1 else "alone") + (" joined" if joined else " split" if S > 1 else ""), (B, T, D, N, G, P, S)
        R = 8 if N <= 8 else 16
        seen.add((R, what))
        d = vlib.VsvSsm(dtype=0, N=N, softplus=1, B=B, T=T, D=D, G=G, x=16, dt=16, b=16, c=16, a=16, y=16)
        assert L.vsv_ssm_scan_ws_bytes(C.byref(d)) == (4 * B * S * (R + 1) * D if S > 1 else 0), (B, T, D, N, G)
    assert seen == {(R, lanes + how) for R in (8, 16) for lanes in ("shared", "alone") for how in ("", " split", " joined")}


def test_c_entries_check_their_arguments():
    from vsv import lib as vlib
    L = vlib.load()
    conv = lambda **k: vlib.VsvShortConv(**{**dict(dtype=0, K=4, silu=1, B=1, T=4, D=8, x=16, x_bs=32, x_ts=8, w=16, y=16), **k})    # noqa: E731
    scan = lambda **k: vlib.VsvSsm(**{**dict(dtype=0, N=4, softplus=1, B=1, T=4, D=8, G=1, x=16, dt=16, b=16, c=16, a=16, y=16), **k})   # noqa: E731
    for bad in (conv(K=0), conv(K=5), conv(B=-1), conv(T=-1), conv(D=0), conv(dtype=3), conv(w=None), conv(x=None), conv(y=None)):
        assert L.vsv_short_conv(C.byref(bad), None) == -1 and L.vsv_last_error()
        assert L.vsv_short_conv_backward(C.byref(bad), None, None, 0, None) == -1
    assert L.vsv_short_conv(None, None) == -1
    g = vlib.VsvShortConvGrads(dy=16, dx=16)
    assert L.vsv_short_conv_backward(C.byref(conv()), C.byref(g), None, 0, None) == -1 and b"workspace" in L.vsv_last_error()
    assert L.vsv_short_conv_step(C.byref(conv()), None) == -1                                  # (no state)
    for bad in (scan(x_ts=2**26), scan(gate=16, gate_ts=-1), scan(D=2**26)):
        assert L.vsv_ssm_scan(C.byref(bad), None, 0, None) == -2 and b"stride" in L.vsv_last_error()
    for bad in (scan(N=0), scan(N=17), scan(G=3), scan(G=0), scan(B=-1), scan(T=-1), scan(D=0), scan(dtype=-1), scan(a=None), scan(x=None),
                scan(c=None), scan(y=None)):
        assert L.vsv_ssm_scan(C.byref(bad), None, 0, None) == -1 and L.vsv_last_error()
        assert L.vsv_ssm_scan_backward(C.byref(bad), None, None, 0, None) == -1
    s = vlib.VsvSsmGrads(dy=16, dx=16, ddt=16, db=16, dc=16)
    assert L.vsv_ssm_scan_backward(C.byref(scan()), C.byref(s), 16, 1 << 30, None) == -1       # (nothing saved)
    assert L.vsv_ssm_scan_backward(C.byref(scan(saved=16)), C.byref(s), None, 0, None) == -1 and b"workspace" in L.vsv_last_error()
    assert L.vsv_ssm_step(C.byref(scan()), None) == -1                                         # (no state)
    row = (C.c_uint64 * 7)(16, 16, 16, 16, 0, 0, 4)
    ok = (1e-3, 0.9, 0.999, 1e-8, 0.01, 1)
    for bits, hyper in ((16, ok), (8, ok), (32, (-1.0,) + ok[1:]), (32, ok[:1] + (1.0,) + ok[2:]), (32, ok[:5] + (0,)), (32, (float("nan"),) + ok[1:])):
        assert L.vsv_adamw_multi(row, 1, 0, bits, *hyper, None) == -1, (bits, hyper)
    assert L.vsv_adamw_multi(row, 1, 3, 32, *ok, None) == -1
    assert L.vsv_adamw_multi(None, 1, 0, 32, *ok, None) == -1
    assert L.vsv_adamw_multi((C.c_uint64 * 7)(0, 16, 16, 16, 0, 0, 4), 1, 0, 32, *ok, None) == -1
    assert L.vsv_adamw_read8(row, 1, None) == -1
    assert L.vsv_adamw_multi(None, 0, 0, 32, *ok, None) == 0                                   # nothing to do
