"""GPU: AdamW over many tensors (moments in 32 and 8 bits), the global gradient norm and the rows of
8-bit moments against their definitions in 64 bits (tests/optim_oracle.py, whose bounds count the
32-bit roundings)."""
import copy
import math

import numpy as np
import pytest
import torch

import optim_oracle as orc
from own_process import own_process  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = (0, 1, 2, 3, 63, 64, 255, 256, 257, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 33333)
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def optim():
    from gsr import optim
    return optim


def cuda(t, offset=0):
    """t on the GPU, `offset` elements into a larger allocation (odd alignments)."""
    store = torch.zeros(t.numel() + offset + 5, dtype=t.dtype, device=DEV)
    out = store[offset:offset + t.numel()].view(t.shape)
    out.copy_(t)
    return out


def raw(t):
    return t.detach().reshape(-1).view(torch.uint8)


def gradients(shape, g, kind=torch.float32, zeros=0.3):
    x = torch.randn(shape, generator=g) * torch.exp(2.0 * torch.randn(shape, generator=g)) * 1e-3
    return (x * (torch.rand(shape, generator=g) > zeros)).to(kind)


def make(optim, shapes, kind="fp32", grad_kind=None, bits=32, step=7, seed=3, offset=0, fresh=False, **kw):
    """An AdamW over parameters of the shapes with moments as after `step` steps, and CPU copies of
    everything: [(param, grad, master, exp_avg, exp_avg_sq in 64 bits)]."""
    g = torch.Generator().manual_seed(seed)
    params, before = [], []
    opt = None
    for shape in shapes:
        p = cuda(torch.randn(shape, generator=g).to(TYPES[kind]), offset)
        gk = TYPES[grad_kind or kind]
        if gk != p.dtype:
            p.grad_dtype = gk
        p.grad = cuda(gradients(shape, g, gk), offset)
        params.append(p)
    groups = [{"params": [p], "lr": 10.0 ** -(2 + i % 3)} for i, p in enumerate(params)]
    opt = optim.AdamW(groups, moment_bits=bits, seed=seed, **kw)
    for p in params:
        shape = tuple(p.shape)
        st = {"step": torch.full((), step, dtype=torch.int64, device=DEV) if kw.get("capturable") else step}
        if fresh:
            m = v = torch.zeros(shape)
        else:
            m, v = gradients(shape, g) * 0.3, gradients(shape, g) ** 2
        if bits == 32:
            st["exp_avg"], st["exp_avg_sq"] = cuda(m, offset), cuda(v, offset)
            m64, v64 = m.double(), v.double()
        else:
            e = optim.moments8_encode(m.to(DEV), v.to(DEV))
            st.update(zip(e._fields, (cuda(t.view(torch.uint8), offset).view(t.dtype) if t.dtype == optim.CODE else t
                                      for t in e)))
            m64 = orc.value(e.exp_avg, e.exp_avg_scale).view(shape)
            v64 = orc.value(e.exp_avg_root, e.exp_avg_root_scale).view(shape) ** 2
        if kind != "fp32":
            st["master"] = cuda(p.cpu().float() + 2.0 ** -12 * torch.rand(shape, generator=g), offset)
        opt.state[p] = st
        before.append((p.cpu().clone(), p.grad.cpu().clone(), (st["master"] if "master" in st else p).cpu().clone(),
                       m64, v64))
    return opt, params, before


def check(opt, params, before, bits=32, step=7, scale=1.0, eps=1e-8, weight_decay=1e-2, seed=3, first=0):
    for i, (p, (_, g, w, m, v)) in enumerate(zip(params, before), first):
        st = opt.state[p]
        lr = opt.param_groups[i]["lr"]
        (p2, m2, v2), (ep, em, ev) = orc.adamw(w, g, m, v, step=step + 1, lr=float(lr), eps=eps, weight_decay=weight_decay,
                                               scale=scale)
        if bits == 8:  # the moments that enter are a product code * scale (and its square)
            extra = 3 * orc.U
            em, ev = em + extra * m.abs(), ev + 2 * extra * v
            ep = ep * 2
        got = st["master"] if "master" in st else p
        d = (orc.f64(got) - p2).abs() - ep
        assert d.numel() == 0 or float(d.max()) <= 0, (i, tuple(p.shape), float(d.max()))
        if "master" in st:
            assert torch.equal(p.cpu(), st["master"].cpu().to(p.dtype))
        if bits == 32:
            for t, x, e in ((st["exp_avg"], m2, em), (st["exp_avg_sq"], v2, ev)):
                assert t.numel() == 0 or float(((orc.f64(t) - x).abs() - e).max()) <= 0, (i, tuple(p.shape))
        else:
            um, ur = orc.draws(p.numel(), seed, i, step + 1)
            orc.check_codes(st["exp_avg"], st["exp_avg_scale"], m2, em, um)
            r2 = v2.sqrt()
            er = torch.minimum(ev / r2.clamp_min(1e-300), ev.sqrt()) + orc.U * r2
            orc.check_codes(st["exp_avg_root"], st["exp_avg_root_scale"], r2, er, ur, root=True)


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("kind,grad_kind", (("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp32"),
                                            ("fp16", "fp32"), ("fp32", "bf16")))
@pytest.mark.parametrize("offset", (0, 1))
def test_step_over_odd_sizes(optim, bits, kind, grad_kind, offset):
    opt, params, before = make(optim, [(n,) for n in SIZES], kind, grad_kind, bits, offset=offset)
    opt.step()
    check(opt, params, before, bits)
    assert all(opt.state[p]["step"] == 8 for p in params)


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("step", (0, 1, 999, 200000))
def test_step_counts_rates_and_scale(optim, bits, step):
    opt, params, before = make(optim, [(5, 3), (300, 4), (2, 3, 50), ()], bits=bits, step=step, fresh=step == 0,
                               eps=1e-15, weight_decay=0.1)
    opt.step(grad_scale=0.25)
    check(opt, params, before, bits, step=step, scale=0.25, eps=1e-15, weight_decay=0.1)


@pytest.mark.parametrize("bits", (32, 8))
def test_more_tensors_than_one_launch_holds(optim, bits):
    shapes = [(1 + (37 * i) % 700,) for i in range(150)]
    shapes[41] = shapes[42] = shapes[149] = (0,)
    opt, params, before = make(optim, shapes, bits=bits, max_grad_norm=0.05)
    opt.step()
    n, c = orc.norm([b[1] for b in before], max_norm=0.05)
    assert c < 1 and abs(float(opt.grad_norm[0]) - n) <= 4 * orc.U * n
    check(opt, params, before, bits, scale=float(opt.grad_norm[1]))


@pytest.mark.parametrize("bits", (32, 8))
def test_more_tensors_than_one_list_holds(optim, bits):
    opt, params, before = make(optim, [(1 + i % 5,) for i in range(4200)], bits=bits)
    opt.step()
    check(opt, params[4000:], before[4000:], bits, first=4000)
    check(opt, params[:100], before[:100], bits)


@pytest.mark.parametrize("bits", (32, 8))
def test_one_norm_over_groups_of_other_betas(optim, bits):
    """Groups that are stepped apart (their betas differ) are clipped by one norm."""
    opt, params, before = make(optim, [(3000,), (50, 3)], bits=bits, max_grad_norm=0.01)
    opt.param_groups[1]["betas"] = (0.8, 0.99)
    opt.step()
    n, c = orc.norm([b[1] for b in before], max_norm=0.01)
    assert c < 1 and abs(float(opt.grad_norm[0]) - n) <= 4 * orc.U * n
    check(opt, params[:1], before[:1], bits, scale=float(opt.grad_norm[1]))
    (p2, _, _), (ep, _, _) = orc.adamw(before[1][2], before[1][1], *before[1][3:], step=8, lr=1e-3, betas=(0.8, 0.99),
                                       weight_decay=1e-2, scale=float(opt.grad_norm[1]))
    assert float(((orc.f64(params[1]) - p2).abs() - 2 * ep).max()) <= 0


@pytest.mark.parametrize("bits", (32, 8))
def test_a_kept_list_follows_what_changes(optim, bits):
    """100 tensors over steps: the table in memory is written once, and again when gradients are
    others, of another type, when rates part tensors that shared them, or when there are more than
    the 64 that a launch takes; on another stream; after a change of seed."""
    opt, params, before = make(optim, [(1 + (91 * i) % 3000,) for i in range(100)], bits=bits)
    pick = [0, 41, 42, 63, 64, 99]

    def now():
        out = []
        for i in pick:
            p, st = params[i], opt.state[params[i]]
            if bits == 32:
                m, v = st["exp_avg"].cpu().double(), st["exp_avg_sq"].cpu().double()
            else:
                m = orc.value(st["exp_avg"], st["exp_avg_scale"])
                v = orc.value(st["exp_avg_root"], st["exp_avg_root_scale"]) ** 2
            out.append((None, p.grad.cpu().clone(), p.detach().cpu().clone(), m, v))
        return out

    def step(expect_written):
        was, image = now(), None if opt._plans is None else opt._plans[0].image.copy()
        t = int(opt.state[params[0]]["step"])
        opt.step()
        if image is not None:
            assert (opt._plans[0].image == image).all() != expect_written
        for i, b in zip(pick, was):
            check(opt, params[i:i + 1], [b], bits, step=t, first=i, seed=opt.seed)
    step(True)
    step(False)
    step(False)
    for p in params:
        p.grad = p.grad * 0.5  # other addresses
    step(True)
    step(False)
    for g in opt.param_groups:
        g["lr"] = g["lr"] * 0.5  # another rate, shared by the same tensors
    step(False)
    opt.param_groups[41]["lr"] = 0.07
    step(True)
    step(False)
    half = params[63].grad.bfloat16()
    params[63].grad = None
    params[63].grad_dtype = torch.bfloat16
    params[63].grad = half
    step(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(False)  # the same contents, in memory of that stream's own
        assert opt._plans[0].kept_on == s.cuda_stream
    torch.cuda.current_stream().wait_stream(s)
    opt.seed = 5
    step(True)
    for i, g in enumerate(opt.param_groups):
        g["lr"] = 1e-3 + 1e-5 * i  # 100 rates: this step's list is its own
    step(False)
    for g in opt.param_groups:
        g["lr"] = 1e-3
    step(True)
    step(False)


def test_long_lists_without_a_workspace(optim):
    """gsr_adamw_step over 100 tensors with and without the list in memory: the same bits."""
    from gsr import _lib
    made = [make(optim, [(1 + (91 * i) % 5000,) for i in range(100)], bits=8) for _ in range(2)]
    for opt, params, _ in made:
        opt.step()
    a, b = made[0][0], made[1][0]
    a.step()
    plan = b._plans[0]
    plan.desc["step"] = plan.steps + 1
    assert _lib.lib().gsr_adamw_step(100, plan.at, 8, 0.9, 0.999, 1e-8, 3, 1.0, -1.0, None, None, None, None,
                                     _lib.stream_of(plan.device)) == 0
    for p, q in zip(made[0][1], made[1][1]):
        assert torch.equal(p, q) and torch.equal(raw(a.state[p]["exp_avg"]), raw(b.state[q]["exp_avg"]))


@pytest.mark.parametrize("bits", (32, 8))
def test_a_norm_that_is_not_finite_changes_nothing(optim, bits):
    for bad in (math.inf, -math.inf, math.nan):
        for capturable in (False, True):
            opt, params, _ = make(optim, [(300,), (1000,)], bits=bits, max_grad_norm=1.0, capturable=capturable)
            params[0].grad[7] = bad
            was = [{k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in opt.state[p].items()} for p in params]
            ps = [p.clone() for p in params]
            opt.step()
            assert not math.isfinite(float(opt.grad_norm[0]))
            for p, q, old in zip(params, ps, was):
                assert torch.equal(p, q)
                for k, v in old.items():
                    if k == "step":
                        assert int(opt.state[p][k]) == int(v) + (0 if capturable else 1)
                    else:
                        assert torch.equal(opt.state[p][k].view(torch.uint8), v.view(torch.uint8)), k


def test_gradients_that_are_not_finite_stay_in_their_elements(optim):
    """Without clipping a NaN or infinite gradient makes its own parameter and moments NaN (as
    torch's) and leaves the rest of its block of 256 as it is without it."""
    opt, params, _ = make(optim, [(512,)], bits=8)
    ref, rparams, _ = make(optim, [(512,)], bits=8)
    keep = torch.ones(512, dtype=torch.bool)
    for i, bad in ((3, math.nan), (300, math.inf)):
        params[0].grad[i] = bad
        rparams[0].grad[i] = 0.0
        keep[i] = False
    # the reference run's own element must not be its block's largest
    for o, p in ((opt, params[0]), (ref, rparams[0])):
        for k in ("exp_avg", "exp_avg_root"):
            o.state[p][k].view(torch.uint8)[[3, 300]] = 0
    opt.step()
    ref.step()
    a, b = opt.state[params[0]], ref.state[rparams[0]]
    for k in ("exp_avg", "exp_avg_root"):
        assert torch.equal(a[k].view(torch.uint8).cpu()[keep], b[k].view(torch.uint8).cpu()[keep])
        assert bool(torch.isnan(a[k].float().cpu()[~keep]).all())
        assert torch.equal(a[k + "_scale"], b[k + "_scale"])
    assert torch.equal(params[0].cpu()[keep], rparams[0].cpu()[keep])
    assert not bool(torch.isfinite(params[0].cpu()[~keep]).any())


@pytest.mark.parametrize("size", (1e-30, 1e-18, 1.0, 1e15, 3e37))
def test_extreme_gradients_in_8_bits(optim, size):
    """First steps on gradients of any size: the root's square may leave 32 bits, the update may
    not become larger than the formula allows."""
    g = torch.Generator().manual_seed(1)
    p = cuda(torch.zeros(700))
    p.grad = cuda(torch.randn(700, generator=g) * size)
    opt = optim.AdamW([p], lr=1e-3, moment_bits=8, weight_decay=0.0, eps=1e-15)
    opt.step()
    m = 0.1 * orc.f64(p.grad)
    orc.check_codes(opt.state[p]["exp_avg"], opt.state[p]["exp_avg_scale"], m, 4 * orc.U * m.abs(),
                    orc.draws(700, 0, 0, 1)[0])
    if size < 1e18 and size > 1e-17:
        d = p.detach().cpu().double() + 1e-3 * torch.sign(m)
        assert float(d.abs().max()) <= 16 * orc.U * 1e-3
    assert bool(torch.isfinite(p).all())


@pytest.mark.parametrize("size", (2e19, 4e20, 6e20, 3e38))
@pytest.mark.parametrize("bits", (32, 8))
def test_gradients_whose_squares_leave_32_bits(optim, bits, size):
    """|g| from 2^64 on, whose square is no 32-bit number, though (1 - b2) g g or its root may be one.  In 8 bits the
    root is what is held, and 32 bits hold it for every finite g; a v of 32 bits beyond them is infinite (as
    torch's) and its parameter stands still.  An ordinary step follows: nothing becomes NaN."""
    g = torch.Generator().manual_seed(1)
    n = 700
    x = torch.randn(n, generator=g)
    x[5], x[300], x[699] = size, -size, size
    big = torch.zeros(n, dtype=torch.bool)
    big[[5, 300, 699]] = True
    p = cuda(torch.zeros(n))
    opt = optim.AdamW([p], lr=1e-3, moment_bits=bits, weight_decay=0.0, eps=1e-15)
    zero = torch.zeros(n, dtype=torch.float64)
    want = [zero, zero, zero]
    for t in (1, 2):
        p.grad = cuda(x)
        (p2, m2, v2), (ep, em, ev) = orc.adamw(*(want[:1] + [x] + want[1:]), step=t, lr=1e-3, eps=1e-15)
        opt.step()
        st = opt.state[p]
        if t == 1 and bits == 8:
            um, ur = orc.draws(n, 0, 0, 1)
            orc.check_codes(st["exp_avg"], st["exp_avg_scale"], m2, em, um)
            r = v2.sqrt()
            orc.check_codes(st["exp_avg_root"], st["exp_avg_root_scale"], r, 12 * orc.U * r, ur, root=True)
        if bits == 32:
            there = v2 < 2.0 ** 127
            assert float(((orc.f64(st["exp_avg_sq"]) - v2).abs() - ev)[there].max()) <= 0
            assert bool((orc.f64(st["exp_avg_sq"])[~there] == math.inf).all())
            if t == 1:
                assert float(((orc.f64(p) - p2).abs() - ep)[there].max()) <= 0
                assert bool((p.cpu()[~there] == 0).all())
        assert bool(torch.isfinite(p).all())
        # |m| / sqrt(v) is at most 3.2 from the second step on; 8 bits change either by an eighth and more
        assert float(p.abs().max()) <= 1e-3 * t * 8
        want = [p2, m2, v2]
        if bits == 32:  # what the kernel holds
            want = [orc.f64(p), orc.f64(st["exp_avg"]), orc.f64(st["exp_avg_sq"])]
        else:
            assert bool(torch.isfinite(st["exp_avg_root"].float()).all()) and bool((st["exp_avg_root"].float().cpu()[big] > 0).all())
        x = torch.randn(n, generator=g)


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("eps", (1e-30, 1e-38, 1e-40, 1e-44, 1e-60))
def test_the_least_eps_divides_nothing_by_nothing(optim, bits, eps):
    """Elements that never had a gradient stay where they are for every eps above 0, however small: 0 / eps is 0."""
    p = cuda(torch.ones(600))
    x = torch.zeros(600)
    x[::7] = 1.0
    p.grad = cuda(x)
    opt = optim.AdamW([p], lr=1e-3, eps=eps, weight_decay=0.0, moment_bits=bits)
    opt.step()
    got = p.cpu()
    assert bool((got[x == 0] == 1).all()) and float((got[x != 0] - (1 - 1e-3)).abs().max()) <= 4 * orc.U


def test_a_root_never_vanishes(optim):
    """Gradients over twelve orders of magnitude in one block, most of them 0 in a step: r = 0 only
    where there never was a gradient, so m / (sqrt(v) + eps) is never m / eps."""
    n = 256 * 64
    g = torch.Generator().manual_seed(2)
    p = cuda(torch.zeros(n))
    opt = optim.AdamW([p], lr=1.0, weight_decay=0.0, eps=1e-15, moment_bits=8)
    seen = torch.zeros(n, dtype=torch.bool)
    for t in range(1, 40):
        x = torch.randn(n, generator=g) * 10.0 ** (-12 * torch.rand(n, generator=g))
        x *= torch.rand(n, generator=g) < 0.1
        seen |= x != 0
        p.grad = cuda(x)
        opt.step()
        st = opt.state[p]
        assert torch.equal(st["exp_avg_root"].float().cpu() > 0, seen)
        assert not bool((st["exp_avg"].float().cpu()[~seen] != 0).any())
    assert not bool(seen.all())
    assert bool(torch.isfinite(p).all())


def test_the_expected_code_is_the_value(optim):
    """A moment that moves by far less than a step is followed on average: 2^16 elements held at
    v = 1 whose gradient falls to 0.  After T steps E[r] = sqrt(0.999^T).  r is 224 and a little
    less of 448 steps of its block's scale, where a step is 16: a rounding's deviation is at most
    half of it, 1/28 of r, and T of them add in squares; six deviations of the mean."""
    n, T = 256 * 256, 60
    p = cuda(torch.zeros(n))
    opt = optim.AdamW([p], lr=0.0, moment_bits=8, weight_decay=0.0)
    m, v = torch.zeros(n), torch.full((n,), 1.0)
    v[::256] = 4.0  # holds each block's scale
    opt.state[p] = {"step": 1000, **optim.moments8_encode(m.to(DEV), v.to(DEV))._asdict()}
    g = torch.zeros(n)
    g[::256] = 2.0
    p.grad = cuda(g)
    for _ in range(T):
        opt.step()
    r = optim.moments8_decode([opt.state[p][k] for k in optim.Moments8._fields])[1].sqrt()
    r = r.cpu().view(-1, 256)[:, 1:].double()
    want = math.sqrt(0.999 ** T)
    assert abs(float(r.mean()) - want) <= 6 / 28 / math.sqrt(r.numel()) * math.sqrt(T)
    assert float(r.std()) > 0


def test_many_steps_of_8_bits_against_32(optim):
    """2500 steps on the same stationary gradients with moments in 8 and in 32 bits (b2 = 0.999, c = 0.001, scales of
    elements equal).  A root r that was rounded last step is a code, so this step it is off one by d = c / 2 |g^2 / v - 1|
    of itself and, its block's scale moving likewise, by the difference of two such, E = c / 2 * 4 / pi; rounding
    it up or down by a step s adds a variance of d s, and s is r / 16 to r / 8: S = 4e-5 to 8e-5 r^2 a step.
    E[r] is kept and E[r^2] grows by S, which v forgets with c: v is too large by S / c, 4 to 8 %; r's deviation
    decays by b2 a step, so its variance is S / (1 - b2^2): 14 to 20 %.  m is rounded at a random place of its step:
    s^2 / 6 / (1 - 0.81), at most 12 % of m.  The update is off by both, at most 24 %; parts of a block far below its
    largest value are held more coarsely and are not measured here.  Means over 2^16 elements: 4 % on top for
    what is drawn, the 1 % by which E[1 / r] is more than 1 / E[r] and r's own spread (1.6 %)."""
    n = 1 << 16
    g = torch.Generator(device=DEV).manual_seed(11)
    made = []
    for bits in (32, 8):
        p = torch.zeros(n, device=DEV)
        made.append((p, optim.AdamW([p], lr=1.0, weight_decay=0.0, eps=1e-15, moment_bits=bits)))
    total, moved = 0.0, None
    for t in range(2500):
        x = torch.randn(n, generator=g, device=DEV)
        for p, opt in made:
            p.zero_()  # the update alone
            p.grad = x
            opt.step()
        if t >= 2000 and t % 50 == 0:
            a, b = made[0][0].double(), made[1][0].double()
            total += float(((a - b).norm() / a.norm())) / 10
            moved = (a, b)
    st = made[1][1].state[made[1][0]]
    v = optim.moments8_decode([st[k] for k in optim.Moments8._fields])[1].double()
    ratio = v / made[0][1].state[made[0][0]]["exp_avg_sq"].double()
    assert 1.0 <= float(ratio.mean()) <= 1.08 + 0.04
    root = ratio.sqrt()
    assert 0.10 <= float(root.std()) <= 0.20 + 0.04
    assert abs(float(root.mean()) - 1) <= 0.04 + 0.01
    assert total <= 0.24 + 0.04
    # the signs, and the sizes on average, are the exact update's
    a, b = moved
    assert abs(float((a * b).sum() / (a * a).sum()) - 1) <= 0.05


def test_against_torch_over_steps(optim):
    """The reference's optimizer: one group per attribute, Adam with eps 1e-15 (gaussian_model.py:
    259-274), over 20 steps: the two round differently, by about U of a step's size each time."""
    g = torch.Generator().manual_seed(5)
    shapes = [(1001, 3), (1001, 4), (1001, 1), (1,), (32, 256)]
    a = [torch.randn(s, generator=g).to(DEV).requires_grad_() for s in shapes]
    b = [t.detach().clone().requires_grad_() for t in a]
    groups = lambda ps: [{"params": [p], "lr": 10.0 ** -(i + 1), "name": str(i)} for i, p in enumerate(ps)]  # noqa: E731
    ours = optim.AdamW(groups(a), lr=0.0, eps=1e-15, weight_decay=0.0)
    ref = torch.optim.Adam(groups(b), lr=0.0, eps=1e-15)
    for t in range(20):
        for p, q in zip(a, b):
            p.grad = gradients(p.shape, g, zeros=0.0).to(DEV)
            q.grad = p.grad.clone()
        ours.step()
        ref.step()
    for i, (p, q) in enumerate(zip(a, b)):
        # each step is at most 8 lr here; its error 20 U of that and a rounding of p
        bound = 20 * (8 * 10.0 ** -(i + 1) * 20 * orc.U + 2 * orc.U * float(q.detach().abs().max()))
        assert float((p - q).detach().abs().max()) <= bound


def test_parameters_and_gradients_of_a_tape(optim):
    """step() marks the parameters as changed: a backward over a graph that saved them raises."""
    p = torch.randn(10, device=DEV, requires_grad=True)
    opt = optim.AdamW([p], lr=0.1)
    loss = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_strided_and_expanded_gradients(optim):
    opt, params, before = make(optim, [(30, 40)])
    g = params[0].grad.clone()
    params[0].grad = g.t().contiguous().t()
    assert not params[0].grad.is_contiguous()
    opt.step()
    check(opt, params, before)
    opt, params, before = make(optim, [(30, 40)])
    params[0].grad = torch.full((1, 1), 0.5, device=DEV).expand(30, 40)
    opt.step()
    before = [(before[0][0], torch.full((30, 40), 0.5)) + before[0][2:]]
    check(opt, params, before)


def test_parameters_without_gradients_and_zero_grad(optim):
    opt, params, before = make(optim, [(100,), (200,), (300,)], bits=8)
    held = params[1].grad
    params[1].grad = None
    keep = params[1].detach().clone()
    opt.step()
    assert torch.equal(params[1], keep) and opt.state[params[1]]["step"] == 7
    check(opt, [params[0]], [before[0]], 8)
    params[1].grad = held
    params[0].grad = params[2].grad = None
    opt.step()
    assert [opt.state[p]["step"] for p in params] == [8, 8, 8]
    i, p = 1, params[1]
    um, _ = orc.draws(200, 3, i, 8)
    (_, m2, _), (_, em, _) = orc.adamw(before[1][2], before[1][1], *before[1][3:], step=8, lr=1e-3)
    orc.check_codes(opt.state[p]["exp_avg"], opt.state[p]["exp_avg_scale"], m2, em + 3 * orc.U * before[1][3].abs(), um)
    opt.zero_grad()
    opt.step()  # nothing to do
    assert [opt.state[p]["step"] for p in params] == [8, 8, 8]


def test_runs_repeat_bit_for_bit(optim):
    out = []
    for _ in range(2):
        opt, params, _ = make(optim, [(5000,), (77, 3)], bits=8, max_grad_norm=0.1)
        for _ in range(5):
            opt.step()
        out.append([p.clone() for p in params] + [opt.state[p][k].view(torch.uint8) for p in params
                                                  for k in optim.Moments8._fields])
    assert all(torch.equal(x, y) for x, y in zip(*out))


# ---- streams, graphs

@pytest.mark.parametrize("bits", (32, 8))
def test_another_stream(optim, bits):
    opt, params, before = make(optim, [(100000,), (777,)], bits=bits, max_grad_norm=0.2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt.step()
    torch.cuda.current_stream().wait_stream(s)
    check(opt, params, before, bits, scale=float(opt.grad_norm[1]))


@pytest.mark.parametrize("shapes", ([(700,), (64, 3), (5,)], [(1 + 7 * i,) for i in range(70)]))
@pytest.mark.parametrize("bits", (32, 8))
def test_captured_steps(optim, bits, shapes):
    """Two graphs over two optimizers, each replayed several times in turn with eager work between:
    every replay is the eager step, its step count and learning rate being read on the device."""
    made = []
    for seed in (3, 4):
        opt, params, _ = make(optim, shapes, bits=bits, seed=seed, capturable=True, max_grad_norm=0.1)
        twin, tparams, _ = make(optim, shapes, bits=bits, seed=seed, capturable=True, max_grad_norm=0.1)
        lr = torch.tensor(1e-2, device=DEV)
        opt.param_groups[0]["lr"] = lr
        made.append((opt, params, twin, tparams, lr))
    for opt, params, twin, tparams, lr in made:  # a warm-up step each
        twin.param_groups[0]["lr"] = lr.clone()
        opt.step()
        twin.step()
    torch.cuda.synchronize()
    graphs = []
    for opt, *_ in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        graphs.append(graph)
    for k in range(4):
        for graph, (opt, params, twin, tparams, lr) in zip(graphs, made):
            rate = 10.0 ** -(k + 1)
            lr.fill_(rate)
            twin.param_groups[0]["lr"].fill_(rate)
            for p, q in zip(params, tparams):
                p.grad.mul_(0.9)
                q.grad.mul_(0.9)
            graph.replay()
            twin.step()
            junk = torch.randn(1000, device=DEV).sum()  # eager allocations between the replays
            for p, q in zip(params, tparams):
                assert torch.equal(p, q)
                for key in twin.state[q]:
                    assert torch.equal(raw(opt.state[p][key]), raw(twin.state[q][key])), key
            assert torch.equal(opt.grad_norm, twin.grad_norm)
            del junk
            torch.cuda.synchronize()
        assert int(made[0][0].state[made[0][1][0]]["step"]) == 9 + k


def test_captured_clipping_and_rows(optim):
    """The norm, clipping in place and a selection of rows in one graph, replayed on new contents."""
    ps = [torch.zeros(n, device=DEV) for n in (100000, 7, 513)]
    for p in ps:
        p.grad = torch.ones_like(p)
    m = optim.moments8_zeros((1000, 3), DEV)
    ix = torch.arange(1200, device=DEV) - 100
    optim.clip_grad_norm_(ps, 1.0)
    optim.moments8_rows([m], [ix])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim.clip_grad_norm_(ps, 1.0)
        rows, = optim.moments8_rows([m], [ix])
    for k in range(4):
        for p in ps:
            p.grad.normal_()
        e = optim.moments8_encode(torch.randn(1000, 3, device=DEV), torch.rand(1000, 3, device=DEV))
        for x, y in zip(m, e):
            raw(x).copy_(raw(y))
        ix.copy_(torch.randint(-5, 1000, (1200,), device=DEV))
        was = [p.grad.clone() for p in ps]
        norm_and_coef, want = optim.grad_norm(was, 1.0), optim.moments8_rows([e], [ix])[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, norm_and_coef[0])
        assert all(torch.equal(p.grad, g * norm_and_coef[1]) for p, g in zip(ps, was))
        assert all(torch.equal(raw(x), raw(y)) for x, y in zip(rows, want))


def test_two_threads_at_once(optim):
    """Optimizers of two threads, each on its own stream: the steps that each takes alone."""
    import threading

    def steps(made, stream, failed):
        try:
            with torch.cuda.stream(stream):
                for _ in range(20):
                    made[0].step()
                    optim.clip_grad_norm_(made[1], 0.05)
        except Exception as e:  # noqa: BLE001
            failed.append(e)
    shapes = ([(70000,), (33, 5)], [(1 + 9 * i,) for i in range(60)])
    pairs = [[make(optim, sh, bits=8, seed=k, max_grad_norm=0.3) for _ in range(2)] for k, sh in enumerate(shapes)]
    torch.cuda.synchronize()
    failed, streams = [], [torch.cuda.Stream() for _ in pairs]
    threads = [threading.Thread(target=steps, args=(pair[0], s, failed)) for pair, s in zip(pairs, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for pair, s in zip(pairs, streams):
        steps(pair[1], s, failed)
    torch.cuda.synchronize()
    assert not failed
    for (opt, params, _), (twin, tparams, _) in pairs:
        for p, q in zip(params, tparams):
            assert torch.equal(p, q) and torch.equal(p.grad, q.grad)
            assert all(torch.equal(raw(torch.as_tensor(opt.state[p][k])), raw(torch.as_tensor(twin.state[q][k]))) for k in twin.state[q])


def test_capture_is_refused_where_it_could_not_be_replayed(optim):
    opt, params, _ = make(optim, [(700,)])
    opt.step()
    was = params[0].detach().clone()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    fresh = optim.AdamW(params, capturable=True)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.step()
    low = torch.zeros(10, dtype=torch.bfloat16, device=DEV)
    low.grad = torch.ones_like(low)
    half = optim.AdamW([low], capturable=True)
    half.step()
    del half.state[low]["master"]
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            half.step()
    torch.cuda.synchronize()
    assert torch.equal(params[0], was)


# ---- the norm

@pytest.mark.parametrize("kind", ("fp32", "bf16", "fp16"))
@pytest.mark.parametrize("offset", (0, 1, 3))
def test_norm_and_clipping(optim, kind, offset):
    g = torch.Generator().manual_seed(9)
    ps = []
    for n in SIZES + (70001,):
        p = torch.zeros(n, dtype=TYPES[kind], device=DEV)
        p.grad = cuda(gradients((n,), g, TYPES[kind]), offset)
        ps.append(p)
    ps.append(torch.zeros(3, device=DEV))  # no gradient
    before = [p.grad.cpu().clone() for p in ps[:-1]]
    for limit in (1e9, 0.01):
        n, c = orc.norm(before, max_norm=limit)
        got = optim.grad_norm([p.grad for p in ps[:-1]], limit).cpu().double()
        assert abs(float(got[0]) - n) <= 2 * orc.U * n and abs(float(got[1]) - c) <= 2 * orc.U
        out = optim.clip_grad_norm_(ps, limit)
        assert out.dim() == 0 and abs(float(out) - n) <= 2 * orc.U * n
        if limit > 1:
            assert all(torch.equal(p.grad.cpu(), b) for p, b in zip(ps, before))
        else:
            for p, b in zip(ps, before):
                want = (b.float() * got[1].float()).to(b.dtype)
                assert torch.equal(p.grad.cpu(), want)


@pytest.mark.parametrize("count", (335, 336, 337, 1000))
def test_norm_and_clipping_over_long_lists(optim, count):
    """More tensors than a launch takes, of three types, with empty ones and ends of chunks among them."""
    g = torch.Generator().manual_seed(count)
    ps = []
    for i in range(count):
        n = (0, 1, 8191, 8192, 8193, 16384, 17)[i % 7] if i % 3 else 1 + 37 * i % 9000
        p = torch.zeros(n, dtype=list(TYPES.values())[i % 3], device=DEV)
        p.grad = cuda(gradients((n,), g, p.dtype), i % 2)
        ps.append(p)
    was = [p.grad.cpu() for p in ps]
    want = math.sqrt(sum(float((w.double() ** 2).sum()) for w in was))
    norm_and_coef = optim.grad_norm([p.grad for p in ps], 0.1)
    assert abs(float(norm_and_coef[0]) - want) <= 2 * orc.U * want
    norm = optim.clip_grad_norm_(ps, 0.1)
    assert torch.equal(norm, norm_and_coef[0])
    coef = norm_and_coef[1].cpu()
    for p, w in zip(ps, was):
        assert torch.equal(p.grad.cpu(), (w.float() * coef).to(w.dtype))


def test_norm_extremes(optim):
    big = torch.full((1000,), 3e38, device=DEV)
    assert abs(float(optim.grad_norm([big[:1]])[0]) / 3e38 - 1) < 1e-6
    assert math.isinf(float(optim.grad_norm([big])[0]))  # beyond float32
    tiny = torch.full((1000,), 1e-40, device=DEV)
    want = math.sqrt(1000) * float(tiny[0].double())
    assert abs(float(optim.grad_norm([tiny])[0].double()) - want) <= 2.0 ** -149
    assert float(optim.grad_norm([torch.empty(0, device=DEV)], 1.0)[0]) == 0.0
    assert float(optim.grad_norm([torch.empty(0, device=DEV)], 1.0)[1]) == 1.0
    got = optim.grad_norm([torch.full((4,), 2.0, device=DEV)], 1.0, grad_scale=-0.5)
    assert float(got[0]) == 2.0 and abs(float(got[1]) - 0.5) < 1e-6
    p = torch.zeros(4, device=DEV)
    p.grad = torch.tensor([1.0, math.inf, 0.0, -2.0], device=DEV)
    ref = torch.zeros(4, device=DEV)
    ref.grad = p.grad.clone()
    n, m = optim.clip_grad_norm_([p], 1.0), torch.nn.utils.clip_grad_norm_([ref], 1.0)
    assert torch.equal(n, m) and torch.equal(torch.isnan(p.grad), torch.isnan(ref.grad))
    assert torch.equal(p.grad.nan_to_num(7.0), ref.grad.nan_to_num(7.0))
    with pytest.raises(RuntimeError, match="not finite"):
        p.grad.fill_(math.nan)
        optim.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert float(optim.clip_grad_norm_([torch.zeros(3, device=DEV)], 1.0)) == 0.0


def test_clipping_strided_gradients_in_place(optim):
    p = torch.zeros(20, 30, device=DEV)
    p.grad = torch.randn(30, 20, device=DEV).t()
    g, at = p.grad.clone(), p.grad.data_ptr()
    optim.clip_grad_norm_(p, 0.5)
    assert p.grad.data_ptr() == at and not p.grad.is_contiguous()
    assert torch.allclose(p.grad, g * (0.5 / g.norm()), rtol=1e-5)


def test_clipping_refuses_what_it_could_not_scale_once(optim):
    p = torch.zeros(20, device=DEV)
    p.grad = torch.ones(20, device=DEV)
    with pytest.raises(ValueError, match="twice"):
        optim.clip_grad_norm_([p, p], 0.5)
    q = torch.zeros(20, 3, device=DEV)
    q.grad = torch.ones(1, 1, device=DEV).expand(20, 3)
    with pytest.raises(ValueError, match="expanded"):
        optim.clip_grad_norm_([p, q], 0.5)
    assert bool((p.grad == 1).all())


def test_refusals_of_the_optimizer(optim):
    p = torch.zeros(20, device=DEV)
    p.grad = torch.ones(20, device=DEV)
    for bad, error in ((dict(lr=-1.0), ValueError), (dict(betas=(0.9, 1.0)), ValueError), (dict(eps=-1.0), ValueError),
                       (dict(weight_decay=-1.0), ValueError), (dict(lr=torch.tensor(0.1, device=DEV)), ValueError)):
        with pytest.raises(error):
            optim.AdamW([p], **bad)
    with pytest.raises(TypeError, match="float64"):
        optim.AdamW([p.double()])
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([torch.zeros(4, 5, device=DEV).t()])
    with pytest.raises(ValueError, match="share memory"):
        q = p[5:10]
        q.grad = torch.ones(5, device=DEV)
        optim.AdamW([p, q]).step()
    opt = optim.AdamW([p])
    with pytest.raises(TypeError):
        opt.add_param_group({"params": [torch.zeros(3, dtype=torch.int32, device=DEV)]})
    assert len(opt.param_groups) == 1
    opt.step()
    was = p.clone()
    for key, bad, error in (("exp_avg", torch.zeros(19, device=DEV), ValueError),
                            ("exp_avg", torch.zeros(20, device=DEV, dtype=torch.float16), ValueError),
                            ("exp_avg_sq", torch.zeros(20), RuntimeError), ("exp_avg", torch.zeros(40, device=DEV)[::2], ValueError)):
        good = opt.state[p][key]
        opt.state[p][key] = bad
        with pytest.raises(error):
            opt.step()
        opt.state[p][key] = good
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError, match="lr"):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-3
    p.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.tensor([1.0]), (20,), device=DEV)
    with pytest.raises(ValueError, match="dense"):
        opt.step()
    assert torch.equal(p, was) and int(opt.state[p]["step"]) == 1
    opt8 = optim.AdamW([p], moment_bits=8)
    p.grad = torch.ones(20, device=DEV)
    opt8.state[p] = opt.state[p]
    with pytest.raises(ValueError, match="8-bit"):
        opt8.step()
    m = optim.moments8_zeros((10, 3), DEV)
    for bad in ((m.exp_avg, m.exp_avg_root, m.exp_avg_scale), (m.exp_avg.float(),) + m[1:],
                (m.exp_avg[:5],) + m[1:], m[:2] + (m.exp_avg_scale[:0], m.exp_avg_root_scale)):
        with pytest.raises((ValueError, TypeError)):
            optim.moments8_decode(bad)
    for ix in (torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(3, 1, dtype=torch.int64, device=DEV),
               torch.zeros(6, dtype=torch.int64, device=DEV)[::2]):
        with pytest.raises(ValueError, match="index"):
            optim.moments8_rows([m], [ix])
    with pytest.raises(ValueError, match="replace_rows"):
        opt.replace_rows([torch.zeros(3, device=DEV)], [p], [torch.arange(3, device=DEV)])
    with pytest.raises(ValueError, match="index"):
        opt.replace_rows([p], [torch.zeros(3, device=DEV)], [torch.arange(4, device=DEV)])


def test_what_changes_in_place_is_seen_or_refused(optim):
    """Betas in a list, options set after construction, states that share a step count, overlapping and
    negated gradients."""
    p = torch.zeros(20, device=DEV)
    p.grad = torch.ones(20, device=DEV)
    opt = optim.AdamW([p], betas=[0.9, 0.999])
    opt.step()
    assert opt.param_groups[0]["betas"] == (0.9, 0.999)
    opt.param_groups[0]["betas"] = [0.5, 0.999]
    opt.step()
    with pytest.raises(TypeError):
        opt.param_groups[0]["betas"][0] = 0.25
    assert opt._plans[0].betas == (0.5, 0.999)
    for name in ("moment_bits", "capturable"):
        with pytest.raises(AttributeError):
            setattr(opt, name, 8)
    opt.max_grad_norm = -1.0
    with pytest.raises(ValueError, match="max_grad_norm"):
        opt.step()
    opt.max_grad_norm = 1.0
    opt.step()
    assert int(opt.state[p]["step"]) == 3 and float(opt.grad_norm[0]) == np.float32(20 ** 0.5)

    q = torch.zeros(20, device=DEV)
    q.grad = torch.ones(20, device=DEV)
    both = optim.AdamW([p, q], capturable=True)
    both.step()
    both.state[q]["step"] = both.state[p]["step"]
    with pytest.raises(ValueError, match="share memory"):
        both.step()

    pool = torch.ones(30, device=DEV)
    p.grad, q.grad = pool[:20], pool[10:]
    with pytest.raises(ValueError, match="share memory"):
        optim.clip_grad_norm_([p, q], 0.5)
    assert bool((pool == 1).all())

    a, b = torch.zeros(20, device=DEV), torch.zeros(20, device=DEV)
    a.grad, b.grad = torch._neg_view(torch.ones(20, device=DEV)), -torch.ones(20, device=DEV)
    for x in (a, b):
        one = optim.AdamW([x])
        one.step()
        one.step()
    assert torch.equal(a, b) and bool((a > 0).all())
    assert float(optim.clip_grad_norm_([a], 1.0)) == np.float32(20 ** 0.5)
    assert torch.equal(a.grad.resolve_neg(), b.grad * optim.grad_norm([b.grad], 1.0)[1])


def test_a_strided_gradient_twice_is_refused(optim):
    p = torch.zeros(4, 5, device=DEV)
    p.grad = torch.ones(5, 4, device=DEV).t()
    with pytest.raises(ValueError, match="twice"):
        optim.clip_grad_norm_([p, p], 0.5)
    assert bool((p.grad == 1).all())


def test_a_refused_state_dict_changes_nothing(optim):
    p = torch.ones(20, device=DEV)
    p.grad = torch.ones(20, device=DEV)
    opt = optim.AdamW([p], lr=0.1)
    opt.step()
    good, st = copy.deepcopy(opt.state_dict()), dict(opt.state[p])
    short = copy.deepcopy(good)
    short["state"][0]["exp_avg"] = torch.zeros(19, device=DEV)
    rate = copy.deepcopy(good)
    rate["param_groups"][0]["lr"] = -1.0
    none = copy.deepcopy(good)
    none["state"][0] = {"step": 3}
    for bad in (short, rate, none):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]["lr"] == 0.1 and all(opt.state[p][k] is v for k, v in st.items())
    opt.load_state_dict(good)
    opt.step()
    assert int(opt.state[p]["step"]) == 2


def test_a_state_or_a_parameter_that_was_replaced_is_used(optim):
    """What the table was made of can change between steps: p.data, a state's tensor, its step, the
    whole state, a group's betas; the next step goes by what is there."""
    opt, params, before = make(optim, [(300,), (40,)])
    opt.step()
    p = params[0]
    m, v = torch.full((300,), 0.5, device=DEV), torch.full((300,), 0.25, device=DEV)
    opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"] = m, v
    opt.state[p]["step"] = 99
    p.data = torch.ones(300, device=DEV)
    opt.param_groups[0]["lr"] = 0.02
    now = [(None, before[0][1], p.detach().cpu().clone(), m.cpu().double(), v.cpu().double())]
    opt.step()
    check(opt, [p], now, step=99)
    assert int(opt.state[p]["step"]) == 100 and int(opt.state[params[1]]["step"]) == 9
    opt.param_groups[0]["betas"] = (0.5, 0.9)
    opt.param_groups[1]["weight_decay"] = 0.0
    st = opt.state[p]
    was = (p.detach().cpu().clone(), st["exp_avg"].cpu().double(), st["exp_avg_sq"].cpu().double())
    opt.step()
    (p2, m2, v2), (ep, em, ev) = orc.adamw(was[0], before[0][1], was[1], was[2], step=101, lr=0.02, betas=(0.5, 0.9),
                                           weight_decay=1e-2)
    assert float(((orc.f64(p) - p2).abs() - ep).max()) <= 0
    assert float(((orc.f64(opt.state[p]["exp_avg"]) - m2).abs() - em).max()) <= 0


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("kind", ("bf16", "fp16"))
def test_a_16_bit_parameter_that_the_program_writes_is_kept(optim, bits, kind):
    """Weights that the program puts into a 16-bit parameter between steps (a loaded model, a clamp, an average, a new
    p.data) are what the next step starts from; where the parameter is its master's rounding the master stays."""
    writes = (lambda p, x: p.copy_(x), lambda p, x: p[:100].copy_(x[:100]), lambda p, x: p.clamp_(-0.5, 0.5),
              lambda p, x: setattr(p, "data", x.clone()), lambda p, x: p.mul_(1.0))
    for write in writes:
        opt, params, _ = make(optim, [(300,), (40,)], kind, bits=bits, weight_decay=0.0)
        opt.step()
        p, st = params[0], opt.state[params[0]]
        x = torch.randn(300, device=DEV).to(p.dtype)
        master = st["master"].clone()
        with torch.no_grad():
            write(p, x)
        want = torch.where(master.to(p.dtype) == p, master, p.float())
        other = opt.state[params[1]]["master"].clone()
        before = [(None, q.grad.cpu(), w.cpu()) for q, w in zip(params, (want, other))]
        moments = [[t.clone() for t in (opt.state[q][k] for k in optim._names(bits)[:-2])] for q in params]
        opt.step()
        for k, (q, (_, g, w), m) in enumerate(zip(params, before, moments)):
            if bits == 8:
                m, v = orc.value(m[0], m[2]), orc.value(m[1], m[3]) ** 2
            else:
                m, v = (t.cpu().double() for t in m)
            check(opt, [q], [(None, g, w, m, v)], bits, step=8, weight_decay=0.0, first=k)
    # a parameter that had no gradient meanwhile, and one step without it
    opt, params, _ = make(optim, [(300,), (40,)], kind, bits=bits, weight_decay=0.0)
    opt.step()
    p, g = params[0], params[0].grad
    p.grad = None
    with torch.no_grad():
        p.fill_(2.0)
    opt.step()
    assert bool((p == 2).all())
    p.grad = g
    m = [opt.state[p][k].clone() for k in optim._names(bits)[:-2]]
    m, v = (orc.value(m[0], m[2]), orc.value(m[1], m[3]) ** 2) if bits == 8 else (t.cpu().double() for t in m)
    opt.step()
    check(opt, [p], [(None, g.cpu(), torch.full((300,), 2.0), m, v)], bits, step=8, weight_decay=0.0)


def test_a_loaded_master_stays_with_its_parameter(optim):
    """The optimizer's state before the model's weights, or behind them: the masters' lower bits survive both; weights
    of another model do not lose to the masters."""
    p = torch.randn(300, device=DEV).bfloat16()
    p.grad = torch.randn(300, device=DEV).bfloat16()
    opt = optim.AdamW([p], lr=1e-4, weight_decay=0.0)
    for _ in range(3):
        opt.step()
    saved, weights = copy.deepcopy(opt.state_dict()), p.clone()
    opt.step()
    want, wanted = opt.state[p]["master"].clone(), p.clone()
    for first in (True, False):
        q = torch.zeros_like(p)
        q.grad = p.grad
        twin = optim.AdamW([q])
        if first:
            twin.load_state_dict(saved)
        with torch.no_grad():
            q.copy_(weights)
        if not first:
            twin.load_state_dict(saved)
        twin.step()
        assert torch.equal(twin.state[q]["master"], want) and torch.equal(q, wanted)
    twin.load_state_dict(saved)
    with torch.no_grad():
        q.fill_(8.0)
    twin.step()
    assert float((twin.state[q]["master"] - 8).abs().max()) <= 1e-3


def test_masters_in_a_captured_step(optim):
    """A parameter that is written before the capture, and between replays through masters_from_parameters()."""
    p = torch.zeros(300, dtype=torch.bfloat16, device=DEV)
    p.grad = torch.zeros_like(p)
    opt = optim.AdamW([p], capturable=True, weight_decay=0.0)
    opt.step()
    p.fill_(2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for value in (2.0, 3.0, 4.0):
        p.data.fill_(value)  # no version counter tells this
        opt.masters_from_parameters()
        graph.replay()
        torch.cuda.synchronize()
        assert bool((p == value).all()) and bool((opt.state[p]["master"] == value).all())
    opt.step()
    assert bool((p == 4).all())


def test_norm_order_is_fixed(optim):
    g = [torch.randn(n, device=DEV) for n in (100000, 77, 300001)]
    a = optim.grad_norm(g)
    assert all(torch.equal(optim.grad_norm(g), a) for _ in range(5))


# ---- 8-bit moments: conversion and rows

@pytest.mark.parametrize("n", SIZES)
def test_encode_and_decode(optim, n):
    g = torch.Generator().manual_seed(n)
    m, v = gradients((n,), g), gradients((n,), g) ** 2
    e = optim.moments8_encode(m.to(DEV), v.to(DEV))
    zero = torch.zeros(n, dtype=torch.float64)
    orc.check_codes(e.exp_avg, e.exp_avg_scale, m.double(), zero)
    root = v.double().sqrt()
    orc.check_codes(e.exp_avg_root, e.exp_avg_root_scale, root, 2 * orc.U * root, root=True)
    a, b = optim.moments8_decode(e)
    x, r = orc.value(e.exp_avg, e.exp_avg_scale), orc.value(e.exp_avg_root, e.exp_avg_root_scale)
    assert bool(((a.cpu().double() - x).abs() <= orc.U * x.abs()).all())
    assert bool(((b.cpu().double() - r * r).abs() <= 4 * orc.U * r * r + 2.0 ** -149).all())
    again = optim.moments8_encode(a, b)  # what is held stays
    assert torch.equal(again.exp_avg.float(), e.exp_avg.float())


def test_encoding_negated_views(optim):
    """A view whose memory holds its values' negatives is encoded as its values."""
    m, v = torch.randn(600, device=DEV), torch.rand(600, device=DEV)
    want = optim.moments8_encode(m, v)
    got = optim.moments8_encode(torch._neg_view(-m), torch._neg_view(-v))
    assert all(torch.equal(raw(x), raw(y)) for x, y in zip(got, want))


def test_encode_what_is_not_finite(optim):
    m = torch.randn(600)
    v = m * m
    m2, v2 = m.clone(), v.clone()
    for i, bad in ((5, math.nan), (400, math.inf), (401, -math.inf)):
        m2[i] = bad
        v2[i] = abs(bad)
        m[i] = v[i] = 0.0
    a, b = optim.moments8_encode(m2.to(DEV), v2.to(DEV)), optim.moments8_encode(m.to(DEV), v.to(DEV))
    ok = torch.isfinite(m2)
    for k in ("exp_avg", "exp_avg_root"):
        x, y = getattr(a, k).float().cpu(), getattr(b, k).float().cpu()
        assert torch.equal(x[ok], y[ok]) and bool(torch.isnan(x[~ok]).all())
        assert torch.equal(getattr(a, k + "_scale"), getattr(b, k + "_scale"))
    z = optim.moments8_encode(torch.zeros(300, device=DEV), torch.zeros(300, device=DEV))
    assert all(float(t.float().abs().max()) == 0 for t in z)
    t = optim.moments8_encode(torch.full((300,), 1e-40, device=DEV), torch.full((300,), 1e-40, device=DEV))
    assert all(bool(torch.isfinite(x.float()).all()) for x in t)
    assert bool((t.exp_avg_root.float() > 0).all())


@pytest.mark.parametrize("shape", ((1,), (7,), (1000,), (100, 3), (1000, 4), (333, 45), (257, 1), (3, 500), (40, 3, 15)))
def test_rows(optim, shape):
    g = torch.Generator().manual_seed(shape[0])
    e = optim.moments8_encode(gradients(shape, g).to(DEV), (gradients(shape, g) ** 2).to(DEV))
    n = shape[0]
    picks = [torch.arange(n), torch.arange(0), torch.randint(0, n, (2 * n + 3,), generator=g),
             torch.cat([torch.nonzero(torch.rand(n, generator=g) < 0.6).view(-1), torch.full((n // 3 + 1,), -1)]),
             torch.tensor([n, -2, 1 << 40, 0, -(1 << 60), n - 1, n - 1])]
    out = optim.moments8_rows([e] * len(picks), [ix.to(DEV) for ix in picks])
    for ix, new in zip(picks, out):
        assert new.exp_avg.shape == (len(ix),) + shape[1:]
        there = (ix >= 0) & (ix < n)
        for code, scale, root in ((0, 2, False), (1, 3, True)):
            x = orc.value(e[code], e[scale]).view(shape)[torch.where(there, ix, 0)] if len(ix) else torch.zeros(
                (0,) + shape[1:], dtype=torch.float64)
            x = x * there.view(-1, *([1] * (len(shape) - 1)))
            orc.check_codes(new[code], new[scale], x, orc.U * x.abs(), root=root)
    assert torch.equal(out[0].exp_avg.float(), e.exp_avg.float())  # all rows in order: unchanged


def test_rows_of_nothing(optim):
    none = optim.moments8_zeros((0, 3), DEV)
    out = optim.moments8_rows([none, optim.moments8_zeros((4, 0), DEV)],
                              [torch.tensor([-1, 5], device=DEV), torch.tensor([1], device=DEV)])
    assert out[0].exp_avg.shape == (2, 3) and float(out[0].exp_avg.float().abs().sum()) == 0
    assert out[1].exp_avg.shape == (1, 0)
    assert optim.moments8_rows([], []) == []


# ---- states that come from elsewhere

def reference_surgery(opt, keep, extra):
    """What _prune_optimizer and cat_tensors_to_optimizer do to the optimizer's state
    (gaussian_model.py:438-511)."""
    for group in opt.param_groups:
        p = group["params"][0]
        st = opt.state.pop(p)
        more = torch.ones((extra,) + tuple(p.shape[1:]), device=p.device)
        for k in ("exp_avg", "exp_avg_sq"):
            st[k] = torch.cat([st[k][keep], torch.zeros_like(more)])
        group["params"][0] = torch.nn.Parameter(torch.cat([p.detach()[keep], more]))
        opt.state[group["params"][0]] = st


def test_the_references_surgery_works_on_32_bit_states(optim):
    opt, params, before = make(optim, [(100, 3), (100, 1), (100, 4)])
    keep = torch.rand(100, generator=torch.Generator().manual_seed(0)) < 0.5
    opt.step()
    opt.step()  # the table is made and used
    before = [(None, None, p.detach().cpu(), opt.state[p]["exp_avg"].cpu(), opt.state[p]["exp_avg_sq"].cpu()) for p in params]
    reference_surgery(opt, keep.to(DEV), 5)
    new = [g["params"][0] for g in opt.param_groups]
    g = torch.Generator().manual_seed(8)
    rows = []
    for p, (_, _, w, m, v) in zip(new, before):
        p.grad = gradients(p.shape, g).to(DEV)
        z = torch.zeros((5,) + tuple(p.shape[1:]))
        rows.append((None, p.grad.cpu(), torch.cat([w[keep], z + 1]), torch.cat([m[keep], z]).double(),
                     torch.cat([v[keep], z]).double()))
    opt.step()
    check(opt, new, rows, step=9)


@pytest.mark.parametrize("cols", (1, 2, 3, 4))
def test_rows_that_are_not_finite_stay_in_their_elements(optim, cols):
    """A NaN code is a NaN in the selection; the other elements of its block are held as without it."""
    g = torch.Generator().manual_seed(cols)
    e = optim.moments8_encode(gradients((600, cols), g).to(DEV), (gradients((600, cols), g) ** 2).to(DEV))
    ix = torch.randint(0, 600, (1000,), generator=g).to(DEV)
    bad = [optim.Moments8(*(t.clone() if t.dtype != optim.CODE else t.view(torch.uint8).clone().view(t.dtype) for t in e))
           for _ in range(2)]
    for i, code in ((5, 0x7f), (300, 0xff), (301, 0x7f)):
        for k in range(2):
            bad[0][k].view(torch.uint8)[i, i % cols] = code
            bad[1][k].view(torch.uint8)[i, i % cols] = 0
    a, b = optim.moments8_rows(bad, [ix, ix])
    for k in range(2):
        x, y = a[k].float(), b[k].float()
        nan = torch.isnan(bad[0][k].float())[ix]
        assert torch.equal(torch.isnan(x), nan) and torch.equal(x[~nan], y[~nan]) and torch.equal(a[2 + k], b[2 + k])


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("kind", ("fp32", "bf16"))
def test_replace_rows(optim, bits, kind):
    opt, params, before = make(optim, [(100, 3), (100,), (50, 4)], kind, bits=bits)
    index = [torch.tensor([5, 5, 99, -1, 0], device=DEV), torch.arange(100, device=DEV).flip(0),
             torch.tensor([-1, -1], device=DEV)]
    new = [torch.randn((len(ix),) + tuple(p.shape[1:]), device=DEV).to(p.dtype) for p, ix in zip(params, index)]
    old_states = [dict(opt.state[p]) for p in params]
    opt.replace_rows(params[:2], new[:2], index[:2])
    assert [g["params"][0] is q for g, q in zip(opt.param_groups, new)] == [True, True, False]
    opt.replace_rows([params[2]], [new[2]], [index[2]])
    assert all(p not in opt.state for p in params)
    for q, ix, st, (_, _, w, m, v) in zip(new, index, old_states, before):
        s = opt.state[q]
        ix = ix.cpu()
        mask = (ix >= 0).view(-1, *([1] * (q.dim() - 1)))
        pick = lambda t: torch.where(mask, t[ix.clamp_min(0)], torch.zeros((), dtype=t.dtype))  # noqa: E731
        assert s["step"] == 7
        if bits == 32:
            assert torch.equal(s["exp_avg"].cpu(), pick(st["exp_avg"].cpu()))
            assert torch.equal(s["exp_avg_sq"].cpu(), pick(st["exp_avg_sq"].cpu()))
        else:
            x = pick(m)
            orc.check_codes(s["exp_avg"], s["exp_avg_scale"], x, orc.U * x.abs())
            x = pick(v.sqrt())
            orc.check_codes(s["exp_avg_root"], s["exp_avg_root_scale"], x, 2 * orc.U * x, root=True)
        if kind != "fp32":
            assert torch.equal(s["master"].cpu(), torch.where(mask, w[ix.clamp_min(0)], q.cpu().float()))
        q.grad = torch.ones_like(q)
    opt.step()


def test_what_is_written_into_replaced_rows_is_kept(optim):
    """A 16-bit parameter that replace_rows put in place and the program then writes: the step starts from that; kept
    rows that it leaves alone have their masters' lower bits."""
    opt, params, _ = make(optim, [(100, 3), (20,)], "bf16", weight_decay=0.0)
    opt.step()
    for same in (False, True):
        p = opt.param_groups[0]["params"][0]
        ix = torch.arange(100, device=DEV).flip(0)
        master = opt.state[p]["master"][ix].clone()
        q = p if same else p.detach()[ix].clone()
        with torch.no_grad():
            if same:
                q.copy_(p[ix])
        q.grad = torch.zeros_like(q)
        opt.replace_rows([p], [q], [ix])
        with torch.no_grad():
            q[:50] = 3.0
        st = opt.state[q]
        st["exp_avg"].zero_()  # a step that moves nothing
        opt.step()
        want = torch.where(torch.arange(100, device=DEV).view(-1, 1) < 50, 3.0, master)
        assert torch.equal(st["master"], want) and torch.equal(q.float(), want.to(q.dtype).float())


def test_replace_rows_takes_each_parameter_once(optim):
    """A new parameter that is listed twice, or is another one of the optimizer's, is refused and nothing changes."""
    opt, params, _ = make(optim, [(10, 3), (10, 3)])
    ix = torch.arange(10, device=DEV)
    q = torch.zeros(10, 3, device=DEV)
    for old, new in ((params, [q, q]), (params[:1], [params[1]])):
        with pytest.raises(ValueError, match="replace_rows"):
            opt.replace_rows(old, new, [ix] * len(old))
        assert [g["params"][0] is p for g, p in zip(opt.param_groups, params)] == [True, True]
        assert all(p in opt.state for p in params)
    opt.replace_rows(params, params, [ix, ix.flip(0)])  # in their own places: other rows' moments
    opt.step()


@pytest.mark.parametrize("bits", (32, 8))
def test_state_dicts(optim, bits):
    """Into this optimizer from torch's Adam, from moments of either width, and through copies."""
    g = torch.Generator().manual_seed(0)
    ps = [torch.randn(s, generator=g).to(DEV).requires_grad_() for s in ((300, 3), (7,))]
    ref = torch.optim.Adam(ps, lr=0.01)
    for p in ps:
        p.grad = gradients(p.shape, g).to(DEV)
    ref.step()
    ref.step()
    opt = optim.AdamW(ps, moment_bits=bits)
    opt.load_state_dict(ref.state_dict())
    assert opt.param_groups[0]["lr"] == 0.01 and opt.state[ps[0]]["step"] == 2
    if bits == 32:
        assert all(torch.equal(opt.state[p][k], ref.state[p][k]) for p in ps for k in ("exp_avg", "exp_avg_sq"))
    else:
        e = optim.moments8_encode(ref.state[ps[0]]["exp_avg"], ref.state[ps[0]]["exp_avg_sq"])
        assert all(torch.equal(opt.state[ps[0]][k].view(torch.uint8), t.view(torch.uint8)) for k, t in e._asdict().items())
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    other = optim.AdamW(ps, moment_bits=40 - bits)
    other.load_state_dict(opt.state_dict())
    other.step()
    twin_ps = [p.detach().clone().requires_grad_() for p in ps]
    twin = optim.AdamW(twin_ps, moment_bits=bits)
    twin.load_state_dict(saved)
    for p, q in zip(ps, twin_ps):
        q.grad = p.grad.clone()
        q.data.copy_(p)
    opt.load_state_dict(saved)
    opt.step()
    twin.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, twin_ps))
    assert all(torch.equal(opt.state[p]["exp_avg"].view(torch.uint8), twin.state[q]["exp_avg"].view(torch.uint8))
               for p, q in zip(ps, twin_ps))
    dup = copy.deepcopy(opt)
    assert (dup.moment_bits, dup.seed, dup.max_grad_norm) == (opt.moment_bits, opt.seed, opt.max_grad_norm)
    for p, q in zip(ps, dup.param_groups[0]["params"]):
        q.grad = p.grad.clone()
    dup.step()
    opt.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, dup.param_groups[0]["params"]))


def test_bfloat16_states_survive_a_state_dict(optim):
    p = torch.randn(300, device=DEV).bfloat16().requires_grad_()
    p.grad = torch.randn(300, device=DEV).bfloat16()
    opt = optim.AdamW([p])
    opt.step()
    st = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in opt.state[p].items()}
    opt.load_state_dict(opt.state_dict())
    for k, v in st.items():
        w = opt.state[p][k]
        assert w == v if k == "step" else w.dtype == v.dtype and torch.equal(w, v)


@pytest.mark.parametrize("bits", (32, 8))
def test_hooks_around_load_state_dict_see_the_state(optim, bits):
    """Hooks before a load get the state that is loaded, and what they return is; hooks behind it find it in place."""
    p = torch.randn(300, device=DEV).bfloat16().requires_grad_()
    p.grad = torch.randn(300, device=DEV).bfloat16()
    opt = optim.AdamW([p], moment_bits=bits)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    other = optim.AdamW([p], moment_bits=bits)
    seen = []

    def before(o, sd):
        seen.append(sorted(sd["state"]))
        sd = dict(sd, state={0: dict(sd["state"][0], step=41)})
        return sd
    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(lambda o: seen.append(int(o.state[p]["step"])))
    other.load_state_dict(saved)
    assert seen == [[0], 41] and saved["state"][0]["step"] == 1
    st = other.state[p]
    assert st["master"].dtype == torch.float32 and torch.equal(st["master"], opt.state[p]["master"])
    assert torch.equal(raw(st["exp_avg"]), raw(opt.state[p]["exp_avg"]))
    other.step()
    assert int(other.state[p]["step"]) == 42
    with pytest.raises(ValueError):  # refused by torch: another number of parameters
        other.load_state_dict(dict(saved, param_groups=[dict(saved["param_groups"][0], params=[0, 1])]))
    assert int(other.state[p]["step"]) == 42


@pytest.mark.parametrize("bits", (32, 8))
def test_states_of_other_layouts_are_loaded_as_the_parameters(optim, bits):
    """Codes, moments and masters that were saved flat or transposed are laid out as their parameter; scales that do
    not fit are refused before anything changes."""
    p = torch.randn(40, 15, device=DEV).bfloat16()
    p.grad = torch.randn(40, 15, device=DEV).bfloat16()
    opt = optim.AdamW([p], moment_bits=bits)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    st = saved["state"][0]
    for k in ("exp_avg", "exp_avg_root", "master"):
        if k in st:
            st[k] = st[k].t().contiguous().t() if k == "master" else st[k].reshape(-1)
    other = optim.AdamW([p], moment_bits=bits)
    other.load_state_dict(saved)
    for k, t in opt.state[p].items():
        if k != "step":
            assert torch.equal(raw(other.state[p][k]), raw(t)) and other.state[p][k].shape == t.shape, k
    if bits == 8:
        ix = torch.tensor([3, -1, 39], device=DEV)
        a, b = (optim.moments8_rows([[o.state[p][k] for k in optim.Moments8._fields]], [ix])[0] for o in (opt, other))
        assert all(torch.equal(raw(x), raw(y)) for x, y in zip(a, b))
        st["exp_avg_scale"] = st["exp_avg_scale"][:-1]
        was = dict(other.state[p])
        for o in (other, optim.AdamW([p])):
            with pytest.raises(ValueError):
                o.load_state_dict(saved)
        assert all(other.state[p][k] is v for k, v in was.items())
    other.step()


# ---- nothing outside

class Fenced:
    """Tensors inside larger allocations filled with a pattern; check() finds what was written around them."""

    def __init__(self):
        self.stores = []

    def __call__(self, t, offset=0, align=256):
        size = t.element_size()
        n, at = t.numel() * size, align + offset * size
        store = torch.full((at + n + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        out = store[at:at + n].view(t.dtype).view(t.shape)
        out.copy_(t)
        self.stores.append((store, at, n))
        return out

    def bytes(self, n):
        return self(torch.zeros(n, dtype=torch.uint8))

    def check(self):
        torch.cuda.synchronize()
        for store, at, n in self.stores:
            assert bool((store[:at] == 0xA5).all()) and bool((store[at + n:] == 0xA5).all()), (at, n)


@pytest.mark.parametrize("kind,bits,offset", [(k, b, o) for k in TYPES for b in (32, 8) for o in (0, 1)])
@pytest.mark.parametrize("counted", (False, True))
@pytest.mark.parametrize("sizes", (SIZES, (2000001, 300000), tuple(1 + (331 * i) % 5000 for i in range(130))))
def test_a_step_writes_its_tensors_alone(optim, kind, bits, offset, counted, sizes):
    """Parameters, masters, moments, scales, counts, the norm, the workspace and the kept list."""
    from gsr import _lib
    g, fence, L = torch.Generator().manual_seed(1), Fenced(), _lib.lib()
    desc = np.zeros(len(sizes), optim.STEP_DTYPE)
    T = TYPES[kind]
    for k, n in enumerate(sizes):
        p = torch.randn(n, generator=g).to(T)
        moment = (lambda: fence(torch.rand(n, generator=g), offset)) if bits == 32 else (
            lambda: fence(torch.randint(0, 0x78, (n,), generator=g, dtype=torch.uint8), offset))
        scale = (lambda: fence(torch.rand(-(-n // 256), generator=g) + 0.1).data_ptr()) if bits == 8 else (lambda: 0)
        desc[k] = (fence(p, offset).data_ptr(), fence(gradients((n,), g, T), offset).data_ptr(),
                   fence(p.float(), offset).data_ptr() if kind != "fp32" else 0, moment().data_ptr(), moment().data_ptr(),
                   scale(), scale(), n, 0, 3, fence(torch.tensor([3])).data_ptr() if counted else 0, 0, 1e-3, 1e-2, k,
                   {"fp32": 0, "bf16": 1, "fp16": 2}[kind], {"fp32": 0, "bf16": 1, "fp16": 2}[kind], 0)
    at = desc.ctypes.data
    clip, work = fence(torch.zeros(2)), fence.bytes(L.gsr_adamw_workspace_bytes(len(sizes), at, 1))
    kept = fence.bytes(L.gsr_adamw_kept_bytes(len(sizes)))
    image = np.zeros(1 + 2 * len(sizes), np.int64)
    for max_norm in (0.5, -1.0):
        for keep in (False, True) if kept.numel() else (False,):
            torch.cuda.synchronize()
            assert L.gsr_adamw_step(len(sizes), at, bits, 0.9, 0.999, 1e-8, 0, 1.0, max_norm, clip.data_ptr(),
                                    work.data_ptr(), kept.data_ptr() if keep else None,
                                    image.ctypes.data if keep else None, 0) == 0
            fence.check()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("offset", (0, 1))
def test_the_norm_and_scaling_write_theirs_alone(optim, kind, offset):
    from gsr import _lib
    g, fence, L = torch.Generator().manual_seed(1), Fenced(), _lib.lib()
    sizes = SIZES * 9 + (8191, 8193, 70000001)
    grads = [fence(torch.ones(n).to(TYPES[kind]), offset) for n in sizes]
    desc = np.zeros(len(sizes), optim.GRAD_DTYPE)
    desc["grad"], desc["n"], desc["type"] = [t.data_ptr() for t in grads], sizes, list(TYPES).index(kind)
    at = desc.ctypes.data
    out, work = fence(torch.zeros(2)), fence.bytes(L.gsr_grad_norm_workspace_bytes(len(sizes), at))
    torch.cuda.synchronize()
    assert L.gsr_grad_norm(len(sizes), at, 1.0, 1.0, out.data_ptr(), work.data_ptr(), 0) == 0
    assert L.gsr_grad_scale(len(sizes), at, out.data_ptr(), 0) == 0
    fence.check()
    assert abs(float(out[0]) - math.sqrt(sum(sizes))) <= orc.U * math.sqrt(sum(sizes))


@pytest.mark.parametrize("cols", (1, 2, 3, 4, 5, 7, 16, 45, 255, 256, 257, 1000))
@pytest.mark.parametrize("offset", (0, 1, 3))
def test_rows_write_theirs_alone(optim, cols, offset):
    """The selection ends anywhere; the last source row, whose words reach its end, among what is taken."""
    from gsr import _lib
    g, fence, L = torch.Generator().manual_seed(cols), Fenced(), _lib.lib()
    src, rows = 37, 111
    index = torch.randint(-2, src + 2, (rows,), generator=g)
    index[-1] = src - 1
    desc = np.zeros(1, optim._ROWS_DTYPE)
    codes = [fence(torch.randint(0, 0x78, (src * cols,), generator=g, dtype=torch.uint8), offset) for _ in range(2)]
    scales = [fence(torch.rand(-(-src * cols // 256), generator=g)) for _ in range(2)]
    to = [fence.bytes(rows * cols + offset)[offset:] for _ in range(2)]
    to_scales = [fence(torch.zeros(-(-rows * cols // 256))) for _ in range(2)]
    desc[0] = (*(t.data_ptr() for t in (*codes, *scales, fence(index), *to, *to_scales)), src, rows, cols, 0)
    torch.cuda.synchronize()
    assert L.gsr_moment_rows(1, desc.ctypes.data, 0) == 0
    n = src * cols
    full = [fence(torch.rand(n, generator=g), offset) for _ in range(2)]
    assert L.gsr_moments_decode(n, *(t.data_ptr() for t in (*codes, *scales, *full)), 0) == 0
    assert L.gsr_moments_encode(n, *(t.data_ptr() for t in (*full, *codes, *scales)), 0) == 0
    fence.check()


# ---- long tensors

def test_rows_and_scaling_beyond_32_bits(optim):
    """A source of 2^32 + 48 elements, and a gradient of as many."""
    rows = (1 << 28) + 3
    m = optim.moments8_zeros((rows, 16), DEV)
    for r, code in ((0, 0x38), (rows - 1, 0x40)):  # 1.0 and 2.0
        m.exp_avg.view(torch.uint8)[r] = code
        m.exp_avg_root.view(torch.uint8)[r] = code
        m.exp_avg_scale[r * 16 // 256] = m.exp_avg_root_scale[r * 16 // 256] = 3.0
    new = optim.moments8_rows([m], [torch.tensor([rows - 1, -1, 0, rows, rows - 1], device=DEV)])[0]
    a, b = optim.moments8_decode(new)
    want = torch.tensor([6.0, 0.0, 3.0, 0.0, 6.0])[:, None].expand(5, 16)
    assert torch.allclose(a.cpu(), want, rtol=1e-6) and torch.allclose(b.cpu(), want * want, rtol=1e-6)
    del m
    p = torch.zeros((1 << 32) + 48, dtype=torch.bfloat16, device=DEV)
    p.grad = torch.zeros_like(p)
    at = torch.tensor([0, (1 << 31) + 1, (1 << 32) - 1, (1 << 32) + 47], device=DEV)
    p.grad[at] = torch.tensor([3.0, 4.0, 12.0, 84.0], dtype=torch.bfloat16, device=DEV)
    n = optim.clip_grad_norm_([p], 8.5)
    assert abs(float(n) - 85.0) < 1e-5
    assert torch.allclose(p.grad[at].cpu().float(), torch.tensor([0.3, 0.4, 1.2, 8.4]), rtol=2.0 ** -8)


@pytest.mark.parametrize("bits", (32, 8))
def test_offsets_beyond_32_bits(optim, bits):
    """2^32 + 777 elements: every byte and element offset passes 32 bits.  Zero everywhere but at
    the ends."""
    n = (1 << 32) + 777
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    opt = optim.AdamW([p], lr=0.5, moment_bits=bits, weight_decay=0.0, max_grad_norm=1e9)
    opt.state[p] = opt._new_state(p)
    at = torch.tensor([0, 1, (1 << 31) + 5, (1 << 32) - 1, 1 << 32, (1 << 32) + 300, n - 1], device=DEV)
    p.grad[at] = torch.tensor([1.0, -2.0, 3.0, 4.0, -5.0, 6.0, 7.0], dtype=torch.bfloat16, device=DEV)
    opt.step()
    want = torch.tensor([1.0, -1.0, 1.0, 1.0, -1.0, 1.0, 1.0]) * -0.5
    assert torch.equal(p[at].cpu().float(), want)
    assert abs(float(opt.grad_norm[0]) - math.sqrt(140.0)) <= 4 * orc.U * 12
    assert int(torch.count_nonzero(p[:1 << 31])) + int(torch.count_nonzero(p[1 << 31:])) == 7
    if bits == 8:
        st = opt.state[p]
        m = st["exp_avg"].view(torch.uint8)[at].view(optim.CODE).float() * st["exp_avg_scale"][at // 256]
        assert torch.allclose(m.cpu(), 0.1 * torch.tensor([1.0, -2.0, 3.0, 4.0, -5.0, 6.0, 7.0]), rtol=0.125)
