"""CPU: what AdamW, the norm and the 8-bit moments refuse, before anything reaches the GPU; the
rounding draws' statistics; the oracle's own roundings."""
import ctypes as C

import numpy as np
import pytest
import torch

import optim_oracle as orc


def _lib():
    from gsr import _lib
    return _lib.lib()


def table(**kw):
    from gsr import optim
    d = np.zeros(1, optim.STEP_DTYPE)
    # made-up addresses: every call below is refused before a launch
    d[0] = (1 << 20, 1 << 20, 0, 1 << 20, 1 << 20, 1 << 20, 1 << 20, 4, 0, 1, 0, 0, 1e-3, 0.0, 0, 0, 0, 0)
    for k, v in kw.items():
        d[k] = v
    return d


@pytest.mark.parametrize("bad,bits", (
    (dict(n=-1), 32), (dict(n=(1 << 33) + 1), 32), (dict(first=-256), 32), (dict(param_type=3), 32), (dict(grad_type=-1), 32),
    (dict(param=0), 32), (dict(grad=0), 32), (dict(m=0), 32), (dict(v=0), 8), (dict(ms=0), 8), (dict(vs=0), 8),
    (dict(master=1 << 20), 32), (dict(param_type=1), 32), (dict(first=128), 8), (dict(lr=-1.0), 32),
    (dict(lr=float("nan")), 32), (dict(weight_decay=-0.1), 32), (dict(step=0), 32), (dict(lr_dev=1 << 20), 32),
    (dict(step_dev=1 << 20), 32), ({}, 16)))
def test_adamw_step_refuses(bad, bits):
    d = table(**bad)
    assert _lib().gsr_adamw_step(1, d.ctypes.data, bits, 0.9, 0.999, 1e-8, 0, 1.0, -1.0, None, None, None, None, None) in (-2, -5)
    assert b"gsr_adamw_step" in _lib().gsr_last_error()


def test_adamw_step_refuses_constants_and_mixed_steps():
    d = table()
    for b1, b2, eps in ((1.0, 0.999, 1e-8), (-0.1, 0.999, 1e-8), (0.9, 1.0, 1e-8), (0.9, 0.999, -1.0),
                        (float("nan"), 0.999, 1e-8)):
        assert _lib().gsr_adamw_step(1, d.ctypes.data, 32, b1, b2, eps, 0, 1.0, -1.0, None, None, None, None, None) == -2
    assert _lib().gsr_adamw_step(-1, d.ctypes.data, 32, 0.9, 0.999, 1e-8, 0, 1.0, -1.0, None, None, None, None, None) == -2
    assert _lib().gsr_adamw_step(1, None, 32, 0.9, 0.999, 1e-8, 0, 1.0, -1.0, None, None, None, None, None) == -2
    p = 1 << 20
    for max_norm, clip, work in ((1.0, None, p), (1.0, p, None), (float("nan"), p, p), (1.0, p, p + 8)):
        assert _lib().gsr_adamw_step(1, d.ctypes.data, 32, 0.9, 0.999, 1e-8, 0, 1.0, max_norm, clip, work, None, None, None) == -2
    assert _lib().gsr_adamw_workspace_bytes(1, d.ctypes.data, 0) == 0
    assert _lib().gsr_adamw_workspace_bytes(1, d.ctypes.data, 1) >= 8
    for kept, image in ((p, None), (None, p), (p + 8, p)):
        assert _lib().gsr_adamw_step(1, d.ctypes.data, 32, 0.9, 0.999, 1e-8, 0, 1.0, -1.0, None, None, kept, image, None) == -2
    assert _lib().gsr_adamw_kept_bytes(42) == 0 and _lib().gsr_adamw_kept_bytes(5000) == 0
    assert _lib().gsr_adamw_kept_bytes(100) >= 100 * (88 + 4)
    many = np.concatenate([table(n=5000, step_dev=p)] * 100)
    assert _lib().gsr_adamw_workspace_bytes(100, many.ctypes.data, 1) >= 100 * (16 + 88 + 4) + 8 * 125
    two = np.concatenate([table(step_dev=1 << 20), table()])
    assert _lib().gsr_adamw_step(2, two.ctypes.data, 32, 0.9, 0.999, 1e-8, 0, 1.0, -1.0, None, 1 << 20, None, None, None) == -2


def test_norm_rows_and_conversions_refuse():
    from gsr import optim
    L = _lib()
    p = 1 << 20
    for bad in ((p, -1, 0, 0), (0, 4, 0, 0), (p, 4, 3, 0), (p, (1 << 33) + 1, 0, 0)):
        d = np.zeros(1, optim.GRAD_DTYPE)
        d[0] = bad
        assert L.gsr_grad_norm(1, d.ctypes.data, 1.0, 1.0, p, p, None) < 0
        assert L.gsr_grad_scale(1, d.ctypes.data, p, None) < 0
    d[0] = (p, 4, 0, 0)
    assert L.gsr_grad_norm(1, d.ctypes.data, 1.0, -1.0, p, p, None) == -2
    assert L.gsr_grad_norm(1, d.ctypes.data, 1.0, 1.0, None, p, None) == -2
    assert L.gsr_grad_norm(1, d.ctypes.data, 1.0, 1.0, p, None, None) == -2
    assert L.gsr_grad_scale(1, d.ctypes.data, None, None) == -2
    assert L.gsr_grad_norm_workspace_bytes(1, d.ctypes.data) >= 8
    r = np.zeros(1, optim._ROWS_DTYPE)
    good = dict(src_m=p, src_r=p, src_ms=p, src_rs=p, index=p, m=p, r=p, ms=p, rs=p, src_rows=4, rows=4, cols=3)
    for bad in (dict(src_rows=-1), dict(rows=-1), dict(cols=0), dict(index=0), dict(m=0), dict(rs=0), dict(src_m=0),
                dict(rows=1 << 33), dict(src_rows=1 << 40)):
        for k, v in {**good, **bad}.items():
            r[k] = v
        assert L.gsr_moment_rows(1, r.ctypes.data, None) == -2, bad
    assert L.gsr_moments_encode(-1, p, p, p, p, p, p, None) == -2
    assert L.gsr_moments_encode(4, p, None, p, p, p, p, None) == -2
    assert L.gsr_moments_decode((1 << 33) + 1, p, p, p, p, p, p, None) == -2
    assert L.gsr_moments_decode(4, p, p, p, None, p, p, None) == -2
    assert L.gsr_moments_encode(0, None, None, None, None, None, None, None) == 0


def test_tables_match_the_header():
    """The numpy tables have the C structures' size and order."""
    from gsr import optim

    class Step(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("param", "grad", "master", "m", "v", "ms", "vs")] + [
            (n, C.c_longlong) for n in ("n", "first", "step")] + [(n, C.c_void_p) for n in ("step_dev", "lr_dev")] + [
            (n, C.c_double) for n in ("lr", "weight_decay")] + [(n, C.c_int) for n in ("ordinal", "param_type", "grad_type",
                                                                                      "reserved")]
    assert C.sizeof(Step) == optim.STEP_DTYPE.itemsize
    for n, *_ in Step._fields_:
        assert getattr(Step, n).offset == optim.STEP_DTYPE.fields[n][1]
    assert optim.GRAD_DTYPE.itemsize == 24 and optim._ROWS_DTYPE.itemsize == 96


def test_cpu_tensors_and_bad_options_are_refused():
    from gsr import optim
    p = torch.zeros(4, requires_grad=True)
    with pytest.raises(RuntimeError, match="GPU"):
        optim.AdamW([p])
    with pytest.raises(RuntimeError, match="GPU"):
        optim.grad_norm([p.detach()])
    with pytest.raises(RuntimeError, match="GPU"):
        optim.moments8_encode(p.detach(), p.detach())
    with pytest.raises(RuntimeError, match="GPU"):
        optim.moments8_rows([optim.moments8_zeros((4,), "cpu")], [torch.zeros(1, dtype=torch.int64)])
    with pytest.raises(ValueError, match="8 or 32"):
        optim.AdamW([p], moment_bits=16)
    with pytest.raises(ValueError, match="max_grad_norm"):
        optim.AdamW([p], max_grad_norm=-1.0)
    with pytest.raises(ValueError, match="no gradients"):
        optim.grad_norm([])
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError, match="indices"):
        optim.moments8_rows([], [torch.zeros(1, dtype=torch.int64)])
    assert float(optim.clip_grad_norm_([p], 1.0)) == 0.0  # no gradients


def test_draws_are_uniform_and_unrelated():
    """16-bit draws over 2^18 elements: means within 5 standard errors of 1/2, no correlation beyond
    5 / sqrt(n) between the two moments, neighbours, steps or tensors."""
    n = 1 << 18
    u = {}
    for name, args in (("a", (0, 0, 1)), ("step", (0, 0, 2)), ("tensor", (0, 1, 1)), ("seed", (1, 0, 1))):
        u[name] = [x.double() / 65536 - 0.5 for x in orc.draws(n, *args)]
    for m, r in u.values():
        for x in (m, r):
            assert abs(float(x.mean()) + 0.5 / 65536) <= 5 / (12 * n) ** 0.5
            assert abs(float((x * x).mean()) - 1 / 12) <= 5 * (1 / 180 / n) ** 0.5
    corr = lambda x, y: abs(float((x * y).mean()) * 12)  # noqa: E731
    a_m, a_r = u["a"]
    pairs = [(a_m, a_r), (a_m[1:], a_m[:-1]), (a_r[1:], a_r[:-1]), (a_m[4:], a_m[:-4]), (a_m[256:], a_m[:-256])]
    pairs += [(u[k][j], u["a"][j]) for k in ("step", "tensor", "seed") for j in (0, 1)]
    for x, y in pairs:
        assert corr(x, y) <= 5 / n ** 0.5


def test_oracle_codes_are_torchs():
    """The oracle's table and nearest rounding against torch's own conversion."""
    tab = orc.table()
    assert torch.equal(tab.float().to(torch.float8_e4m3fn).double(), tab) and float(tab[-1]) == 448.0 and len(tab) == 127
    x = torch.randn(256 * 4, generator=torch.Generator().manual_seed(0)).double()
    top = x.view(-1, 256).abs().amax(1, keepdim=True)
    codes = (x.view(-1, 256) / top * 448).float().to(torch.float8_e4m3fn)
    orc.check_codes(codes, (top.view(-1) / 448).float(), x, torch.zeros_like(x))
    with pytest.raises(AssertionError):
        wrong = codes.float()
        wrong[0, 3] = -wrong[0, 3]
        orc.check_codes(wrong.to(torch.float8_e4m3fn), (top.view(-1) / 448).float(), x, torch.zeros_like(x))


def test_flat_buffers_of_8_bit_moments_begin_at_blocks():
    """FlatParams(moment_bits=8) on the CPU: segments and exchange slices begin at blocks of 256."""
    from gsr import dp, train
    fp = train.FlatParams([("a", (5, 3), 0.1), ("b", (300,), 0.2), ("c", (2, 4), 0.3)], "cpu", moment_bits=8)
    assert fp.offsets == [0, 256, 768] and fp.n == 1024 and fp.align == 256 and not hasattr(fp, "exp_avg")
    m = fp.segment_moments("b")
    assert m.exp_avg.shape == (300,) and m.exp_avg_scale.shape == (2,)
    assert fp.segment_moments("c").exp_avg.shape == (2, 4) and fp.segment_moments("c").exp_avg_scale.shape == (1,)
    with pytest.raises(RuntimeError, match="GPU"):
        fp.step()
    for n in (1024 + 500, 5000 * 256 + 13, 255):
        r = dp.exchange_chunks(n, 4, 1, 256)
        assert r[0][0] == 0 and r[-1][1] == n and all(a[1] == b[0] for a, b in zip(r, r[1:]))
        assert all(lo % 256 == 0 for lo, _ in r)


def test_tensors_are_described_and_recognised():
    """libgsr_tensors.so on CPU tensors: five words of each, and what counts as unchanged."""
    from gsr import _lib
    T = _lib.tensors()
    a, b = torch.zeros(6, requires_grad=True), torch.zeros(2, 3, dtype=torch.bfloat16)
    items = [a, b, b.t(), torch.zeros(3, dtype=torch.int64), None, 5, torch.zeros(2, dtype=torch.float64),
             torch.sparse_coo_tensor(torch.tensor([[1]]), torch.tensor([1.0]), (4,))]
    w = np.zeros((len(items), 5), np.int64)
    assert T.gsr_tensors_describe(items, w.ctypes.data) == 0
    assert w[0].tolist() == [a.data_ptr(), 6, 0, -1, 1] and w[1].tolist() == [b.data_ptr(), 6, 1, -1, 1]
    assert w[2, 4] == 0 and w[3, 2] == 4 and w[4, 2] == -2 and w[5, 2] == -3 and w[6, 2] == -1 and w[7, 4] == 0
    assert T.gsr_tensors_describe((a,), w.ctypes.data) == -1
    a.grad = torch.ones(6)
    assert [g is a.grad for g in T.gsr_tensors_grads([b, a])] == [True]
    with pytest.raises(TypeError):
        T.gsr_tensors_grads([a, 3])
    assert T.gsr_tensors_grad_table([a.grad], np.zeros(1, [("x", "3i8")]).ctypes.data) == -1  # no GPU tensor

    class Opt:
        moment_bits = 32
        param_groups = [{"params": [a]}, {"params": [b]}]
        state = {a: {"exp_avg": torch.zeros(6), "exp_avg_sq": torch.zeros(6), "step": torch.tensor(3)}}
    from gsr import optim
    opt = Opt()
    seen = optim._Seen(opt, [a, b], [a.grad, None])
    got = seen.grads(opt)
    assert got[0] is a.grad and got[1] is None and seen.at.tolist() == [a.grad.data_ptr(), 0] and seen.plain.value == 1
    a.grad = torch.ones(6)  # another gradient: the same optimizer
    assert seen.grads(opt)[0] is a.grad and seen.at[0] == a.grad.data_ptr()

    def differs(change, undo):
        change()
        assert seen.grads(opt) is None
        undo()
        assert seen.grads(opt) is not None
    st, m, g = opt.state[a], opt.state[a]["exp_avg"], a.grad
    differs(lambda: st.update(exp_avg=torch.zeros(6)), lambda: st.update(exp_avg=m))
    differs(lambda: st.update(master=torch.zeros(6)), lambda: st.pop("master"))
    data = m.data
    differs(lambda: setattr(m, "data", torch.zeros(6)), lambda: setattr(m, "data", data))
    pd = a.data
    differs(lambda: setattr(a, "data", pd[:5]), lambda: setattr(a, "data", pd))
    differs(lambda: setattr(a, "grad", None), lambda: setattr(a, "grad", g))
    differs(lambda: setattr(b, "grad", torch.zeros_like(b)), lambda: setattr(b, "grad", None))
    differs(lambda: opt.param_groups[1].update(params=[]), lambda: opt.param_groups[1].update(params=[b]))
    differs(lambda: opt.param_groups[1].update(params=[b, a]), lambda: opt.param_groups[1].update(params=[b]))
    differs(lambda: opt.param_groups[1].update(params=[torch.zeros(2, 3)]), lambda: opt.param_groups[1].update(params=[b]))
    differs(lambda: opt.state.update({b: {}}), lambda: opt.state.pop(b))
    differs(lambda: opt.state.update({a: dict(st)}), lambda: opt.state.update({a: st}))


def test_rows_of_other_tensors_are_not_taken():
    """gsr_tensors_moment_rows: CPU tensors, other types, shapes and numbers of tensors give None."""
    from gsr import _lib, optim
    T, desc = _lib.tensors(), np.zeros(2, optim._ROWS_DTYPE)
    m, ix = optim.moments8_zeros((300, 3), "cpu"), torch.zeros(2, dtype=torch.int64)
    for bad in ([*m, ix], [*m, ix.int()], [*m], [None] * 5, [1, *m[1:], ix], [*m, ix] + [*m]):
        assert T.gsr_tensors_moment_rows(bad, desc.ctypes.data) is None
    assert not desc.view(np.uint8).any()
    assert T.gsr_tensors_moment_rows([], desc.ctypes.data) == []


def test_a_negated_view_is_not_dense():
    """A view whose memory holds its values' negatives has to be copied before a kernel reads it."""
    from gsr import _lib, optim
    x = torch._neg_view(torch.ones(5))
    words = np.zeros((1, 5), np.int64)
    _lib.tensors().gsr_tensors_describe([x], words.ctypes.data)
    assert x.is_contiguous() and words[0, 4] == 0
    y = optim._solid(x)
    _lib.tensors().gsr_tensors_describe([y], words.ctypes.data)
    assert words[0, 4] == 1 and torch.equal(y, -torch.ones(5))


def test_overlapping_gradients_are_found():
    from gsr import _lib, optim
    t = np.zeros(4, optim.GRAD_DTYPE)
    t["grad"], t["n"], t["type"] = (96, 0, 64, 32), (2, 8, 0, 16), (0, 0, 0, 1)  # [96, 104), [0, 32), nothing, [32, 64)
    overlap = lambda: _lib.tensors().gsr_tensors_overlap(t.ctypes.data, 4)  # noqa: E731
    assert overlap() == 0
    for k, n in ((1, 9), (3, 17 + 16)):
        was = t["n"][k]
        t["n"][k] = n
        assert overlap() == 1
        t["n"][k] = was
    t["grad"][0] = 0
    assert overlap() == 1


def test_gradients_outside_48_bits_are_refused():
    from gsr import optim
    d = np.zeros(1, optim.GRAD_DTYPE)
    d["grad"], d["n"] = 1 << 50, 4
    assert _lib().gsr_grad_norm(1, d.ctypes.data, 1.0, 1.0, 1 << 20, 1 << 20, None) == -2
    assert _lib().gsr_grad_scale(1, d.ctypes.data, 1 << 20, None) == -2
    assert _lib().gsr_grad_norm_workspace_bytes(1, d.ctypes.data) == 0


def test_tables_are_not_made_of_other_tensors():
    """gsr_tensors_plan refuses CPU tensors and states that lack something; what a step writes may not overlap."""
    from gsr import _lib, optim
    T, d = _lib.tensors(), np.zeros(2, optim.STEP_DTYPE)
    p, names = torch.zeros(5), optim._names(32)
    st = {"exp_avg": torch.zeros(5), "exp_avg_sq": torch.zeros(5), "step": 1}
    places = np.array([7], np.int32)

    def plan(params, states, names, bits, device):
        return T.gsr_tensors_plan(params, states, names, bits, 0, device, places.ctypes.data, d.ctypes.data)
    assert plan([p], [st], names, 32, 0) == 1 and plan([None], [st], names, 32, 0) == 1
    assert plan([p], [[]], names, 32, -1) == 1 and plan([p], [st], names, 8, -1) == 1
    assert plan([p], [{"exp_avg": st["exp_avg"]}], names, 32, -1) == 1
    assert plan([p], [dict(st, exp_avg_sq=torch.zeros(4))], names, 32, -1) == 1
    assert plan([p.double()], [st], names, 32, -1) == 1 and plan([p.bfloat16()], [st], names, 32, -1) == 1
    assert not d.view(np.uint8).any()
    assert plan([p], [st], names, 32, -1) == 0  # device -1: the CPU's, as gsr_tensors_describe says it
    assert (d["param"][0], d["m"][0], d["v"][0], d["n"][0], d["step"][0], d["ordinal"][0], d["step_dev"][0]) == (
        p.data_ptr(), st["exp_avg"].data_ptr(), st["exp_avg_sq"].data_ptr(), 5, 1, 7, 0)

    def overlap(bits, **kw):
        t = np.zeros(1, optim.STEP_DTYPE)
        for k, v in dict(param=4096, m=8192, v=12288, ms=16384, vs=20480, n=300, param_type=1, master=24576, **kw).items():
            t[k] = v
        return T.gsr_tensors_written_overlap(t.ctypes.data, 1, bits)
    assert overlap(32) == 0 and overlap(8) == 0
    assert overlap(32, step_dev=8192 + 1192) == 1 and overlap(8, step_dev=8192 + 296) == 1
    assert overlap(32, step_dev=8192 + 1200) == 0 and overlap(8, step_dev=8192 + 300) == 0
    assert overlap(32, step_dev=16384) == 0 and overlap(8, step_dev=16384) == 1


def test_the_timed_calls_are_there():
    """What perf/operators.py calls of gsr.optim exists, with the arguments that it passes."""
    import ast
    import inspect
    import os

    from gsr import optim
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    with open(path) as f:
        tree = ast.parse(f.read())
    found = set()
    for call in ast.walk(tree):
        if not isinstance(call, ast.Call) or not isinstance(call.func, ast.Attribute):
            continue
        of = call.func.value
        if (isinstance(of, ast.Call) and getattr(of.func, "id", "") == "_optim") or getattr(of, "id", "") == "optim":
            target = getattr(optim, call.func.attr)
            inspect.signature(target).bind(*call.args, **{k.arg: 0 for k in call.keywords})
            found.add(call.func.attr)
    assert found == {"AdamW", "clip_grad_norm_", "moments8_rows"}
