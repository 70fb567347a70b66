"""vsv.optim.AdamW on the GPU: 32 bits against the formulas in 64 with the state carried in float32, 8 bits code by code.

32 bits: m and v round 3 times a step (product, product, sum), so after s steps they are within 3 s + 1 half steps of float32 at the
sum of their absolute terms; the update m / (sqrt(v) / root + eps) adds 8 more and v's error enters by half.  m's terms cancel: its
error is taken at the sum of absolute terms too.  The parameter adds its own rounding (twice in float32, once per step in its type)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SIZES = [(1,), (3, 5), (255,), (256,), (257,), (2048,), (2049, 3), (0,), (64, 100), (5, 1, 3, 3), (100003,)]


def _setup(dtype, bits, sizes=SIZES, seed=0):
    from vsv.optim import AdamW
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(*s, generator=g).to(DT[dtype]).cuda()) for s in sizes]
    return ps, AdamW(ps, state_bits=bits, **HYPER), g


def _grads(ps, g):
    for p in ps:
        p.grad = (torch.randn(p.shape, generator=g) * torch.exp(2 * torch.randn(p.shape, generator=g)) * 1e-2).to(p.dtype).cuda()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_32_bits(dtype):
    ps, opt, g = _setup(dtype, 32)
    ms = [torch.zeros(p.shape).double() for p in ps]
    vs, mags = [m.clone() for m in ms], [m.clone() for m in ms]
    b1, b2 = HYPER["betas"]
    eps32, own = 2.0 ** -24, torch.finfo(DT[dtype]).eps / 2
    for t in range(1, 5):
        _grads(ps, g)
        before = [p.detach().double().cpu() for p in ps]
        opt.step()
        for i, p in enumerate(ps):
            gr = p.grad.double().cpu()
            ms[i], vs[i], mags[i] = b1 * ms[i] + (1 - b1) * gr, b2 * vs[i] + (1 - b2) * gr * gr, b1 * mags[i] + (1 - b1) * gr.abs()
            st = opt.state[p]
            assert ((st["exp_avg"].double().cpu() - ms[i]).abs() <= (3 * t + 1) * eps32 * mags[i] + 1e-38).all()
            assert ((st["exp_avg_sq"].double().cpu() - vs[i]).abs() <= (4 * t + 1) * eps32 * vs[i] + 1e-38).all()
            den = vs[i].sqrt() / math.sqrt(1 - b2 ** t) + HYPER["eps"]
            rate = HYPER["lr"] / (1 - b1 ** t)
            want = before[i] * (1 - HYPER["lr"] * HYPER["weight_decay"]) - rate * ms[i] / den
            tol = own * want.abs() * 1.01 + 3 * eps32 * before[i].abs() + eps32 * rate * ((3 * t + 1) * mags[i] + (2 * t + 10) * ms[i].abs()) / den
            if dtype == "fp16":
                tol += 2.0 ** -25                                            # (half the smallest step below 2^-14)
            assert ((p.detach().double().cpu() - want).abs() <= tol + 1e-38).all()


def _codes(x, table, top, u):
    """The upper of the two codes around x / top in `table` where it lies more than a share u of the way."""
    part = torch.where(top > 0, x / torch.where(top > 0, top, 1.0), 0.0).clamp(max=1.0)
    low = (torch.bucketize(part, table, right=True) - 1).clamp(max=table.numel() - 2)
    share = (part - table[low]) / (table[low + 1] - table[low])
    return low + (share > u).long(), (share - u).abs()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_8_bits(dtype):
    """Scales within a half step of float32 and every code as the definition's (a share within 1e-9 of its threshold may go
    either way: 64-bit arithmetic on both sides); the state that was read is the state the next step starts from."""
    ps, opt, g = _setup(dtype, 8)
    b1, b2 = HYPER["betas"]
    own = torch.finfo(DT[dtype]).eps / 2
    tm, tv = (torch.arange(128).double() / 127) ** 2, (torch.arange(256).double() / 255) ** 4
    for t in range(1, 5):
        _grads(ps, g)
        before = [p.detach().double().cpu() for p in ps]
        old = [[opt.state[p][k].cpu().clone() for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")] if t > 1 else None for p in ps]
        opt.step()
        for i, p in enumerate(ps):
            n = p.numel()
            if n == 0:
                continue
            st, gr = opt.state[p], p.grad.double().cpu().reshape(-1)
            block = torch.arange(n) // 256
            m, v = torch.zeros(n).double(), torch.zeros(n).double()
            if old[i]:
                km, sm, kv, sv = old[i]
                km, kv = km.reshape(-1).long(), kv.reshape(-1).long()
                m, v = (torch.sign(km) * sm.double()[block] * tm[km.abs()]).float().double(), (sv.double()[block] * tv[kv]).float().double()
            m, v = b1 * m + (1 - b1) * gr, b2 * v + (1 - b2) * gr * gr
            u = (((torch.arange(n) * 0xC13FA9A9 % 2**32) + t * 0x91E10DA5) % 2**32).double().add(0.5) / 2**32
            for x, table, name, share in ((m.abs(), tm, "exp_avg", u), (v, tv, "exp_avg_sq", 1 - u)):
                scale = st[name + "_scale"].cpu()
                top = torch.zeros(scale.numel()).double().scatter_reduce_(0, block, x, "amax")
                assert torch.equal(top.float(), scale), (name, (top - scale.double()).abs().max())
                want, near = _codes(x, table, scale.double()[block], share)
                if name == "exp_avg_sq":
                    want = torch.where((want < 1) & (x > 0), 1, want)
                else:
                    want = want * torch.sign(m).long()
                got = st[name].cpu().reshape(-1).long()
                assert ((got == want) | (near < 1e-9)).all(), (name, (got != want).sum())
            rate, root = HYPER["lr"] / (1 - b1 ** t), math.sqrt(1 - b2 ** t)
            den = v.sqrt() / root + HYPER["eps"]
            want = before[i].reshape(-1) * (1 - HYPER["lr"] * HYPER["weight_decay"]) - rate * m / den
            tol = own * want.abs() * 1.01 + 2.0 ** -24 * (3 * before[i].reshape(-1).abs() + 12 * rate * m.abs() / den) + (2.0 ** -25 if dtype == "fp16" else 1e-38)
            assert ((p.detach().double().cpu().reshape(-1) - want).abs() <= tol).all()
    ms, vs = opt.moments()
    for p, m, v in zip(ps, ms, vs):
        st = opt.state[p]
        block = torch.arange(p.numel()) // 256
        k, q = st["exp_avg"].cpu().reshape(-1).long(), st["exp_avg_sq"].cpu().reshape(-1).long()
        assert torch.equal(m.cpu().reshape(-1), (torch.sign(k) * st["exp_avg_scale"].cpu().double()[block] * tm[k.abs()]).float())
        assert torch.equal(v.cpu().reshape(-1), (st["exp_avg_sq_scale"].cpu().double()[block] * tv[q]).float())


def test_8_bits_moments_are_the_formulas_bit_for_bit():
    """The same bfloat16 gradients twice (few mantissas, so sums that lie next to the middle between two float32 scales are common):
    after either step every moment read back equals the formulas in 64 bits, products and sums rounded one by one."""
    from vsv.optim import AdamW
    g = torch.Generator().manual_seed(9)
    n = 256 * 2000 + 77
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    opt = AdamW([p], state_bits=8)
    p.grad = (torch.randn(n, generator=g) * torch.exp(2 * torch.randn(n, generator=g)) * 1e-3).to(torch.bfloat16).cuda()
    gr, block = p.grad.double().cpu(), torch.arange(n) // 256
    tm, tv = (torch.arange(128).double() / 127) ** 2, (torch.arange(256).double() / 255) ** 4
    m, v = torch.zeros(n).double(), torch.zeros(n).double()
    for t in (1, 2):
        opt.step()
        m, v = m * 0.9 + gr * (1 - 0.9), v * 0.999 + gr * gr * (1 - 0.999)
        u = (((torch.arange(n) * 0xC13FA9A9 % 2**32) + t * 0x91E10DA5) % 2**32).double().add(0.5) / 2**32
        new = []
        for x, table, share in ((m, tm, u), (v, tv, 1 - u)):
            top = torch.zeros(2001).double().scatter_reduce_(0, block, x.abs(), "amax").float().double()[block]
            k, near = _codes(x.abs(), table, top, share)
            assert near.min() > 1e-11                                        # (no share of these inputs is closer to its threshold)
            if table is tv:
                k = torch.where((k < 1) & (x > 0), 1, k)
            new.append((torch.sign(x) * top * table[k]).float().double())
        m, v = new
        got_m, got_v = opt.moments()
        assert (got_m[0].double().cpu() != m).sum() == 0 and (got_v[0].double().cpu() != v).sum() == 0


def test_8_bits_do_not_lose_small_changes():
    """v under gradients of one size: after 700 steps its mean over elements is 1 - 0.999^700 = 0.5036 g^2.  A dither that is even over
    steps and elements keeps the mean's error below half a code step (4 / 255 / 2 = 0.8 %); rounding to the nearest code would freeze it."""
    from vsv.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4096, device="cuda"))
    opt = AdamW([p], lr=0.0, state_bits=8)
    p.grad = torch.full_like(p, 0.5)
    p.grad[::256] = 4.0                                                      # (a block's largest: the others sit at codes of 90)
    for _ in range(700):
        opt.step()
    v = opt.moments()[1][0].view(16, 256)[:, 1:].double().mean().item()
    want = 0.25 * (1 - 0.999 ** 700)
    assert abs(v / want - 1) <= 0.5 * 4 / 90, v / want


def test_not_finite_gradients():
    """32 bits: the element alone is lost.  8 bits: its parameter is NaN, its moments and every neighbour are as without it."""
    for bits in (32, 8):
        ps, opt, g = _setup("fp32", bits, [(1000,)])
        qs, other, _ = _setup("fp32", bits, [(1000,)])
        _grads(ps, g)
        qs[0].grad = ps[0].grad.clone()
        opt.step(); other.step()
        _grads(ps, g)
        qs[0].grad = ps[0].grad.clone()
        for i, bad in ((7, float("nan")), (300, float("inf")), (999, float("-inf"))):
            ps[0].grad[i] = bad
            qs[0].grad[i] = 0.0
        opt.step(); other.step()
        rest = torch.ones(1000, dtype=torch.bool, device="cuda")
        rest[[7, 300, 999]] = False
        assert torch.equal(ps[0].detach()[rest], qs[0].detach()[rest])
        assert torch.isnan(ps[0].detach()[~rest]).all()
        m, v = opt.moments()
        assert torch.isfinite(m[0][rest]).all() and torch.isfinite(v[0][rest]).all()
        if bits == 8:
            assert torch.isfinite(m[0]).all() and torch.isfinite(v[0]).all()


def test_extreme_gradients_8_bits():
    """Zeros, values whose squares leave float32's range at either end, and one value in a whole block."""
    from vsv.optim import AdamW
    p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8)
    p.grad = torch.zeros(1024, device="cuda")
    p.grad[256:512] = 1e-30
    p.grad[512:768] = 3e38
    p.grad[800] = 1.0
    opt.step()
    m, v = opt.moments()
    assert (m[0][:256] == 0).all() and (v[0][:512] == 0).all() and torch.isfinite(m[0]).all() and torch.isfinite(v[0]).all()
    assert (p[:256] == 1).all() and (p[768:800] == 1).all() and torch.isfinite(p).all()
    assert abs(p[800].item() - (1 - 1e-3)) < 1e-6 and abs(p[300].item() - 1) < 1e-6


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_and_many_tensors(bits):
    """150 tensors (three launches), among them views that start off 16 bytes: the same as each alone."""
    from vsv.optim import AdamW
    g = torch.Generator().manual_seed(3)
    base = torch.randn(200_000, generator=g).cuda()
    sizes = [(37 * i) % 2900 + 1 for i in range(150)]
    at, ps = 0, []
    for n in sizes:
        ps.append(torch.nn.Parameter(base[at:at + n]))
        at += n
    copies = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    assert any(p.data_ptr() % 16 for p in ps)
    many, each = AdamW(ps, state_bits=bits, **HYPER), [AdamW([c], state_bits=bits, **HYPER) for c in copies]
    guard = base[at:].clone()
    for _ in range(2):
        for p, c in zip(ps, copies):
            p.grad = torch.randn(p.shape, generator=g).cuda()
            c.grad = p.grad.clone()
        many.step()
        for o in each:
            o.step()
    assert all(torch.equal(p, c) for p, c in zip(ps, copies)) and torch.equal(base[at:], guard)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_groups_and_missing_gradients(bits):
    from vsv.optim import AdamW
    g = torch.Generator().manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(300, generator=g).to(t).cuda()) for t in (torch.float32, torch.bfloat16, torch.float32)]
    opt = AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.5, "weight_decay": 0.0}], state_bits=bits, **{k: v for k, v in HYPER.items()})
    for turn in range(3):
        _grads(ps, g)
        if turn == 1:
            ps[1].grad = None
        opt.step()
    assert [opt.state[p]["step"] for p in ps] == [3, 2, 3]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    again = AdamW([{"params": twins[:2]}, {"params": twins[2:]}], state_bits=bits)
    again.load_state_dict(opt.state_dict())
    for p, q in zip(ps, twins):
        for k, v in opt.state[p].items():
            w = again.state[q][k]
            assert (w == v).all() and w.dtype == v.dtype and w.data_ptr() != v.data_ptr() if torch.is_tensor(v) else w == v
    _grads(ps, g)
    for p, q in zip(ps, twins):
        q.grad = p.grad.clone()
    before = ps[0]._version
    opt.step(); again.step()
    assert ps[0]._version > before
    assert all(torch.equal(p, q) for p, q in zip(ps, twins))


@pytest.mark.parametrize("bits", [32, 8])
def test_copies_and_what_does_not_fit(bits):
    """A deep copy steps like the original; a parameter that has changed its size, and saved state of another shape, are refused
    before anything is launched."""
    import copy
    from vsv.optim import AdamW
    p = torch.nn.Parameter(torch.randn(300, device="cuda"))
    opt = AdamW([p], state_bits=bits)
    p.grad = torch.randn_like(p)
    opt.step()
    q, twin = copy.deepcopy((p, opt))
    q.grad = p.grad.clone()
    twin.param_groups[0]["params"][0].grad = p.grad.clone()
    opt.step(); twin.step()
    assert torch.equal(p, twin.param_groups[0]["params"][0]) and twin.state_bits == bits
    big = torch.nn.Parameter(torch.zeros(600, device="cuda"))
    with pytest.raises(ValueError, match="exp_avg"):
        AdamW([big], state_bits=bits).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="bits"):
        AdamW([p], state_bits=40 - bits).load_state_dict(opt.state_dict())
    p.data = torch.zeros(600, device="cuda")
    p.grad = torch.zeros(600, device="cuda")
    with pytest.raises(ValueError, match="shape"):
        opt.step()


def test_closure_scheduler_and_capture():
    from vsv.optim import AdamW
    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    opt = AdamW([p], lr=1.0, weight_decay=0.0)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)

    def closure():
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss
    assert opt.step(closure).item() == 10.0
    sched.step()
    assert torch.allclose(p, torch.zeros_like(p), atol=1e-6) and opt.param_groups[0]["lr"] == 0.5
    p.grad = torch.ones_like(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        x.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    assert opt.state[p]["step"] == 1


def test_a_refused_step_changes_nothing():
    from vsv.optim import AdamW
    p, q = (torch.nn.Parameter(torch.ones(10, device="cuda")) for _ in range(2))
    opt = AdamW([{"params": [p]}, {"params": [q], "lr": 0.5}])
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.param_groups[1]["betas"] = (0.9, 1.0)
    with pytest.raises(ValueError, match="hyper-parameters"):
        opt.step()
    assert opt.state[p]["step"] == 0 and torch.equal(p, torch.ones_like(p)) and not opt.state[p]["exp_avg"].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_model_train_step_takes_it(bits):
    """CVAEMemRand.train_step(x, optimizer) with this optimizer: the parameters after three steps against torch's own AdamW (32 bits:
    to rounding; 8 bits: within a tenth of a step of lr, as codes are 1.6 % apart near a block's largest value and coarser below)."""
    from oracle import vsv_oracle as vo
    from vae.cvae_with_mem_randomized import CVAEMemRand
    from vsv.optim import AdamW
    import numpy as np
    cfg = vo.make_config(5, 3)
    W = vo.init_weights(cfg, 0, 2.0, np.float32)
    g = torch.Generator().manual_seed(2)
    x = {"surface": (0.2 + 0.1 * torch.randn(4, 21, 5, 5, generator=g)).cuda(), "ex_feats": (0.01 * torch.randn(4, 21, 3, generator=g)).cuda()}
    eps = torch.randn(4, 21, 5, generator=g).cuda()
    done = []
    for make in (lambda m: torch.optim.AdamW(m.parameters(), lr=1e-3), lambda m: AdamW(m.parameters(), lr=1e-3, state_bits=bits)):
        model = CVAEMemRand(dict(cfg, device="cuda:0"))
        model.load_state_dict({k: torch.from_numpy(v) for k, v in W.items()}, strict=False)
        model = model.to("cuda:0")
        start = [p.detach().clone() for p in model.parameters()]
        opt = make(model)
        losses = [float(model.train_step(x, opt, _eps=eps)["loss"]) for _ in range(3)]
        done.append(([p.detach() - s for p, s in zip(model.parameters(), start)], losses))
    (want, lw), (got, lg) = done
    a, b = torch.cat([t.reshape(-1) for t in want]), torch.cat([t.reshape(-1) for t in got])
    assert b.abs().max() > 1e-3
    assert ((a - b).norm() / a.norm()).item() <= (2e-3 if bits == 32 else 0.1)
    assert abs(lw[2] - lg[2]) <= 1e-2 * abs(lw[2])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_first_step_under_capture_leaves_no_state(bits):
    """Refused before the moments are made (their zeros would only be recorded): the eager step behind it starts from zero moments, as
    a new optimizer's does, and replays of the graph leave them alone."""
    from vsv.optim import AdamW
    g = torch.Generator().manual_seed(6)
    p = torch.nn.Parameter(torch.randn(1000, generator=g).cuda())
    q = torch.nn.Parameter(p.detach().clone())
    opt, other = AdamW([p], state_bits=bits, **HYPER), AdamW([q], state_bits=bits, **HYPER)
    p.grad = torch.randn(1000, generator=g).cuda()
    q.grad = p.grad.clone()
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        x.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    assert len(opt.state) == 0
    for turn in range(3):
        graph.replay()
        opt.step(); other.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, q), turn
        assert all(torch.equal(a, b) for one, two in zip(opt.moments(), other.moments()) for a, b in zip(one, two)), turn
    assert x[0].item() == 6


def test_continues_a_checkpoint_of_torchs():
    """State of a torch.optim.AdamW after three steps, loaded, then three more of either: the parameters agree to the rounding of
    test_32_bits' bound (3 s + 1 half steps on the moments, s = 6, 8 on the update, 3 and one more a step on the parameter), twice."""
    from vsv.optim import AdamW
    g = torch.Generator().manual_seed(8)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in SIZES]
    theirs = torch.optim.AdamW(ps, **HYPER)
    for _ in range(3):
        _grads(ps, g)
        theirs.step()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = AdamW(qs)
    opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["weight_decay"] == HYPER["weight_decay"]
    for t in range(4, 7):
        _grads(ps, g)
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
        theirs.step(); opt.step()
        for p, q in zip(ps, qs):
            st = theirs.state[p]
            assert opt.state[q]["step"] == t == int(st["step"])
            size = p.detach().abs() + HYPER["lr"] * 10                       # (|m| / sqrt(v) of a few equal shares is below 10)
            assert ((p - q).detach().abs() <= 2.0 ** -24 * 2 * (4 * t + 30) * size).all()
