"""GPU: 8-bit moments, weight decay and gradient clipping in the training step's flat buffer
(gsr.train.FlatParams, train_step) and through densification, against the 64-bit formulas
(tests/optim_oracle.py)."""
import math

import pytest
import torch

import optim_oracle as orc
from own_process import own_process  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def flat(bits, seed=0, decay=False):
    from gsr import train
    spec = [("a", (700, 3), 1e-2), ("b", (1,), 1e-3), ("c", (256,), 3e-3), ("none", (0, 4), 0.1), ("d", (33, 45), 1e-4)]
    fp = train.FlatParams(spec, DEV, moment_bits=bits)
    g = torch.Generator().manual_seed(seed)
    for name, shape, _ in spec:
        fp.load(name, torch.randn(shape, generator=g).to(DEV))
        x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape, generator=g)) * 1e-3
        fp.params[name].grad.copy_(x)
    if decay:
        fp.set_weight_decay("a", 0.1)
        fp.set_weight_decay("d", 0.02)
    return fp


def segments(fp):
    """Per segment: (parameter, gradient, exp_avg, exp_avg_sq in 64 bits) copies."""
    out = []
    for name, shape, off in zip(fp.names, fp.shapes, fp.offsets):
        n = math.prod(shape)
        if fp.moment_bits == 8:
            s = fp.segment_moments(name)
            m, v = orc.value(s.exp_avg, s.exp_avg_scale), orc.value(s.exp_avg_root, s.exp_avg_root_scale) ** 2
        else:
            m, v = (t[off:off + n].cpu().double() for t in (fp.exp_avg, fp.exp_avg_sq))
        out.append((fp.params[name].detach().reshape(-1).cpu().clone(), fp.params[name].grad.reshape(-1).cpu().clone(), m, v))
    return out


def check(fp, before, scale):
    """fp after one step from `before`: parameters and moments within their roundings."""
    for k, (name, (p, g, m, v)) in enumerate(zip(fp.names, before)):
        if p.numel() == 0:
            continue
        (p2, m2, v2), (ep, em, ev) = orc.adamw(p, g, m, v, step=fp.t, lr=fp.lrs[k], eps=fp.eps, scale=scale,
                                               weight_decay=fp.weight_decays[k])
        extra = 0.0 if fp.moment_bits == 32 else 3 * orc.U
        em, ev, ep = em + extra * m.abs(), ev + 2 * extra * v, ep * (1 if fp.moment_bits == 32 else 2)
        d = (orc.f64(fp.params[name]).reshape(-1) - p2).abs() - ep
        assert float(d.max()) <= 0, (name, float(d.max()))
        if fp.moment_bits == 8:
            s = fp.segment_moments(name)
            um, ur = orc.draws(p.numel(), 0, k, fp.t)
            orc.check_codes(s.exp_avg, s.exp_avg_scale, m2, em, um)
            r = v2.sqrt()
            er = torch.minimum(ev / r.clamp_min(1e-300), ev.sqrt()) + orc.U * r
            orc.check_codes(s.exp_avg_root, s.exp_avg_root_scale, r, er, ur, root=True)
        else:
            off = fp.offsets[k]
            for t, x, e in ((fp.exp_avg, m2, em), (fp.exp_avg_sq, v2, ev)):
                assert float(((t[off:off + x.numel()].cpu().double() - x).abs() - e).max()) <= 0, name


@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("clip", (False, True))
@pytest.mark.parametrize("decay", (False, True))
def test_flat_steps(bits, clip, decay):
    fp = flat(bits, decay=decay)
    for _ in range(3):
        before = segments(fp)
        scale = 0.25
        c = None
        if clip:
            n, want = orc.norm([b[1] for b in before], 0.25, 0.01)
            c = fp.grad_norm(0.01, 0.25)
            assert want < 1 and abs(float(c[0]) - n) <= 4 * orc.U * n and abs(float(c[1]) - want) <= 4 * orc.U
            scale *= float(c[1])
        fp.step(0.25, c)
        check(fp, before, scale)
    assert fp.t == 3


@pytest.mark.parametrize("bits", (32, 8))
def test_flat_ranges_are_the_whole_step(bits):
    """step_range over the data-parallel exchange's slices, in any order: the whole step's bits."""
    from gsr import dp
    a, b = flat(bits, decay=True), flat(bits, decay=True)
    for _ in range(2):
        a.step(0.5)
        b.begin_step(0.5)
        for lo, hi in reversed(dp.exchange_chunks(b.n + 100, 7, 1, b.align)):
            b.step_range(lo, hi)
    assert torch.equal(a.flat, b.flat)
    if bits == 8:
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.moments, b.moments))
        b.begin_step()
        for lo, hi in ((128, 512), (0, 300)):
            with pytest.raises(ValueError, match="multiples of 256"):
                b.step_range(lo, hi)
    else:
        assert torch.equal(a.exp_avg, b.exp_avg)


def test_ranks_agree_bit_for_bit(tmp_path):
    """Two processes that exchange their gradients step the 8-bit buffer to the same bytes, whatever slices each
    takes, and to those of one process that adds the two gradients itself."""
    import os
    import socket
    import subprocess
    import sys

    import optim_rank_worker as worker
    here = os.path.dirname(os.path.abspath(__file__))
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(
        [os.path.join(os.path.dirname(here), "relightable3dgaussians-w_amd"), os.environ.get("PYTHONPATH", "")]))
    ranks = [subprocess.Popen([sys.executable, os.path.join(here, "optim_rank_worker.py"), str(r), "2", str(port),
                               str(tmp_path / "digest")], env=env) for r in range(2)]
    try:
        assert [p.wait(timeout=90) for p in ranks] == [0, 0]
    finally:
        for p in ranks:
            p.kill()
    digests = [(tmp_path / f"digest.{r}").read_text() for r in range(2)]
    alone = worker.steps(2, lambda fp, step: worker.gradient(fp, step, 0) + worker.gradient(fp, step, 1), 1)
    assert digests == [alone, alone]


def test_a_plain_step_is_what_it_was():
    """Without decay and clipping the 32-bit step stays gsr_adam_step's."""
    a, b = flat(32), flat(32)
    a.step(0.5)
    nseg, gs = len(b.names), 0.5
    from gsr import _lib
    import ctypes as C
    b.t += 1
    _lib.check(_lib.lib().gsr_adam_step(b.n, nseg, (C.c_longlong * nseg)(*b.ends), (C.c_double * nseg)(*b.lrs), 0.9, 0.999,
                                        1e-15, 1, gs, b.flat.data_ptr(), b.grad.data_ptr(), b.exp_avg.data_ptr(),
                                        b.exp_avg_sq.data_ptr(), _lib.stream_of(b.device)), "gsr_adam_step")
    assert torch.equal(a.flat, b.flat) and torch.equal(a.exp_avg_sq, b.exp_avg_sq)


def test_flat_refusals():
    from gsr import train
    with pytest.raises(ValueError, match="8 or 32"):
        train.FlatParams([("a", (4,), 0.1)], DEV, moment_bits=16)
    fp = flat(8)
    with pytest.raises(ValueError, match="weight_decay"):
        fp.set_weight_decay("a", -1.0)
    with pytest.raises(ValueError, match="clip"):
        fp.step(1.0, torch.zeros(2))
    with pytest.raises(ValueError, match="clip"):
        fp.step(1.0, torch.zeros(3, device=DEV))
    was = fp.flat.clone()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fp.step()
    assert fp.t == 0 and torch.equal(fp.flat, was)


@pytest.fixture
def scene8():
    from gsr import train
    return train.synthetic_relit_scene(3000, 2, 160, 96, 120.0, torch.device(DEV), seed=3, moment_bits=8)


def test_training_iterations_with_8_bit_moments_and_clipping(scene8):
    """train_step(max_grad_norm): the update is the formula's on the gradient that the iteration
    left in the flat buffer, the moments it had before, and the learning rates of its schedule."""
    from gsr import train
    scene, views, gts = scene8
    fp = scene.fp
    for it in range(3):
        before = segments(fp)
        limit = 1e-3
        loss = train.train_step(scene, views, [0, 1], gts, max_grad_norm=limit)
        torch.cuda.synchronize()
        before = [(p, fp.params[n].grad.reshape(-1).cpu().clone(), m, v) for n, (p, _, m, v) in zip(fp.names, before)]
        n, want = orc.norm([b[1] for b in before], 0.5, limit)
        got = scene.grad_norm.cpu().double()
        assert want < 1 and abs(float(got[0]) - n) <= 4 * orc.U * n and abs(float(got[1]) - want) <= 4 * orc.U
        check(fp, before, 0.5 * float(got[1]))
        assert bool(torch.isfinite(loss)) and fp.t == it + 1
    keep = fp.flat.clone()
    train.train_step(scene, views, [0, 1], gts)  # without clipping: 8 bits all the same
    assert fp.t == 4 and not torch.equal(fp.flat, keep) and bool(torch.isfinite(fp.flat).all())


def test_a_gradient_that_is_not_finite_leaves_the_scene(scene8):
    from gsr import train
    scene, views, gts = scene8
    train.train_step(scene, views, [0, 1], gts, max_grad_norm=1.0)
    fp = scene.fp
    was, codes = fp.flat.clone(), [t.view(torch.uint8).clone() for t in fp.moments]
    bad = [gts[0] * math.nan, gts[1]]
    train.train_step(scene, views, [0, 1], bad, max_grad_norm=1.0)
    assert not bool(torch.isfinite(scene.grad_norm[0]))
    assert torch.equal(fp.flat, was) and all(torch.equal(t.view(torch.uint8), c) for t, c in zip(fp.moments, codes))
    train.train_step(scene, views, [0, 1], gts, max_grad_norm=1.0)
    assert not torch.equal(fp.flat, was) and bool(torch.isfinite(fp.flat).all())


def test_densification_moves_8_bit_moments():
    """densify_and_prune on the same scene with moments in 32 and in 8 bits: the same rows; the
    8-bit moments are those of the kept rows, re-blocked (rounded to the nearest), zeros in new rows,
    and the groups that are not per Gaussian keep their bytes; training goes on."""
    from gsr import densify, train
    dev = torch.device(DEV)
    made = []
    for bits in (32, 8):
        scene, views, gts = train.synthetic_relit_scene(3000, 2, 160, 96, 120.0, dev, seed=3, moment_bits=bits)
        made.append((scene, views, gts))
    big, small = made[0][0], made[1][0]
    # one training state for both: the 8-bit scene's after two iterations
    for _ in range(2):
        train.train_step(small, *made[1][1:2], [0, 1], made[1][2])
    g = torch.Generator().manual_seed(1)
    for n in small.fp.names:
        big.fp.load(n, small.fp.params[n].detach())
        m, v = densify_moments(small.fp, n)
        off, k = big.fp.offsets[big.fp.names.index(n)], m.numel()
        big.fp.exp_avg[off:off + k], big.fp.exp_avg_sq[off:off + k] = m.to(dev), v.to(dev)
    P = small.P
    stats = {"xyz_gradient_accum": torch.rand(P, 1, generator=g).to(dev), "denom": torch.ones(P, 1, device=dev),
             "max_radii2D": (torch.rand(P, generator=g) * 30).to(dev)}
    keep_bytes = {n: [t.view(torch.uint8).clone() for t in small.fp.segment_moments(n)] for n in small.global_groups}
    for s in (big, small):
        s.stats = {k: v.clone() for k, v in stats.items()}
        s.fp.t = 2
        densify.densify_and_prune(s, 0.5, 0.1, 5.0, 25.0, generator=torch.Generator(device=dev).manual_seed(7))
    assert small.P == big.P != P and small.fp.moment_bits == 8 and small.fp.t == 2
    for n in big.fp.names:
        assert torch.equal(big.fp.params[n], small.fp.params[n]), n
        off, k = big.fp.offsets[big.fp.names.index(n)], big.fp.params[n].numel()
        s = small.fp.segment_moments(n)
        if n in small.global_groups:
            assert all(torch.equal(t.view(torch.uint8), b) for t, b in zip(s, keep_bytes[n])), n
            continue
        m, v = big.fp.exp_avg[off:off + k].cpu().double(), big.fp.exp_avg_sq[off:off + k].cpu().double()
        orc.check_codes(s.exp_avg, s.exp_avg_scale, m, 2 * orc.U * m.abs())
        r = v.sqrt()
        orc.check_codes(s.exp_avg_root, s.exp_avg_root_scale, r, 4 * orc.U * r, root=True)
    assert float(small.fp.segment_moments("xyz").exp_avg.float().abs().sum()) > 0
    loss = train.train_step(small, made[1][1], [0, 1], made[1][2], max_grad_norm=1.0)
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(small.fp.flat).all()) and small.fp.t == 3


def densify_moments(fp, name):
    """(exp_avg, exp_avg_sq) of one segment in 32 bits."""
    from gsr import optim
    m, v = optim.moments8_decode([t.reshape(-1) for t in fp.segment_moments(name)])
    return m, v


def test_the_run_of_a_reference_loop():
    """The reference's loop with this optimizer in Adam's place: parameters of the Gaussians and the
    MLP in groups (gaussian_model.py:259-274), the fused render and losses, clipping, the step, and
    pruning by replace_rows; two runs from one seed agree bit for bit in what the optimizer decides
    from equal gradients."""
    import types

    import torch.nn.functional as F

    import relit_shade
    from gsr import optim, relit, train
    dev = torch.device(DEV)
    scene, views, gts = train.synthetic_relit_scene(2000, 1, 128, 96, 100.0, dev, seed=5)
    names = ("xyz", "scaling", "rotation", "opacity", "albedo", "roughness", "metalness")
    leaves = {n: scene.fp.params[n].detach().clone().requires_grad_(True) for n in names}
    sky = {n: scene.fp.params[n].detach() for n in ("sky_angles", "sky_radius")}
    opt = optim.AdamW([{"params": [leaves[n]], "lr": 1e-3, "name": n} for n in names], eps=1e-15, weight_decay=0.0,
                      moment_bits=8, max_grad_norm=0.5)
    pipe, bg = types.SimpleNamespace(compute_cov3D_python=False), torch.zeros(3, device=dev)
    losses = []
    for it in range(4):
        p = dict(leaves, **sky)
        pc = types.SimpleNamespace(
            get_xyz=scene.get_xyz(p), get_scaling=torch.exp(p["scaling"]), get_rotation=F.normalize(p["rotation"]),
            get_opacity=torch.sigmoid(p["opacity"]), get_albedo=torch.sigmoid(p["albedo"]),
            get_roughness=torch.sigmoid(p["roughness"]), get_metalness=torch.sigmoid(p["metalness"]),
            get_is_sky=scene.is_sky)
        light = relit_shade.EnvironmentLight(torch.full((25, 3), 0.1, device=dev), sh_degree=4)
        out = relit.render(views[0], pc, light, torch.full((1, 4, 3), 0.1, device=dev), 1, pipe, bg, debug=False)
        loss = train.view_loss(out, gts[0], views[0].sky_mask, views[0].occluders_mask)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        assert bool(torch.isfinite(opt.grad_norm).all())
        if it == 1:  # prune a third of the foreground rows
            n_fg = leaves["xyz"].shape[0]
            keep_fg = torch.nonzero(torch.rand(n_fg, generator=torch.Generator().manual_seed(0)) < 0.67).view(-1).to(dev)
            n_sky = sky["sky_angles"].shape[0]
            keep_all = torch.cat([keep_fg, torch.arange(n_fg, n_fg + n_sky, device=dev)])
            index = {n: keep_fg if n in ("xyz", "albedo", "roughness", "metalness") else keep_all for n in names}
            new = {n: leaves[n].detach()[index[n]].clone().requires_grad_(True) for n in names}
            was = {n: [opt.state[leaves[n]][k].clone() for k in optim.Moments8._fields] for n in names}
            opt.replace_rows([leaves[n] for n in names], [new[n] for n in names], [index[n] for n in names])
            for n in names:
                x = orc.value(was[n][0], was[n][2]).view(leaves[n].shape)[index[n].cpu()]
                st = opt.state[new[n]]
                orc.check_codes(st["exp_avg"], st["exp_avg_scale"], x, orc.U * x.abs())
                assert int(st["step"]) == 2
            leaves = new
            m = scene.is_sky.reshape(-1)[keep_all]
            scene.set_sky_flags(m)
        opt.zero_grad(set_to_none=True)
    assert all(bool(torch.isfinite(x)) for x in losses)
    assert all(int(opt.state[leaves[n]]["step"]) == 4 for n in names)
