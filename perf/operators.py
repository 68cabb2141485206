"""The optimizer's operators as they are timed: AdamW over many tensors with moments in 32 and in 8 bits, the global
gradient norm with clipping, and the row selection that densification does on 8-bit moments.

Every operator has a plain form here (elementary torch operations) and the framework's call; `own` says which one `run`
makes.  The tensors of a case are views of flat buffers, each starting at a multiple of 256 elements: the plain forms
work on the whole buffers, the framework's calls on the list of views, and both return the buffers.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BETAS, SEED, MAX_NORM = (0.9, 0.999), 77, 1.0
BLOCK = 256           # consecutive elements of a tensor that share one scale of an 8-bit moment
TOP = 448.0           # the largest e4m3 value
LEAST = 2.0 ** -100   # a block's largest value counts as at least this much
MIX_A, MIX_B, MASK = 0x9E3779B1, 0xB504F333, 0xFFFFFFFF
# the environment MLP's weights and biases, with a table of 32-float image embeddings (elements, learning rate)
MLP = [(n, 2e-4) for n in (256 * 32, 256, 256 * 256, 256, 128 * 256, 128, 12 * 128, 12, 128 * 128, 128, 75 * 128, 75)]
# a scene's per-Gaussian groups: (columns, which rows, learning rate)
GROUPS = ((3, "fg", 1.6e-4), (3, "fg", 2.5e-3), (1, "all", 5e-2), (3, "all", 1e-3), (4, "all", 1e-3), (1, "fg", 2e-4),
          (1, "fg", 2e-4), (2, "sky", 1.6e-4))


def listed():
    return [
        # the environment MLP and the embeddings of 400 photographs: 13 small tensors, where latency counts
        dict(name="adamw mlp", op="adamw", set="mlp", images=400, dtype="fp32", step=1500, clip=False),
        # a training scene of 1.5M Gaussians with its MLP: the parameters of one training iteration
        dict(name="adamw scene", op="adamw", set="scene", fg=1363637, sky=136363, images=16, dtype="fp32", step=1500,
             clip=False),
        # 300 weights and biases of odd sizes in 16 bits with 32-bit masters, gradients clipped to a norm first
        dict(name="adamw ragged bf16 clip", op="adamw", set="ragged", count=300, low=64, high=2000000, shapes=1,
             dtype="bf16", step=20, clip=True),
        # the very first step of a small scene: moments all zero
        dict(name="adamw first step", op="adamw", set="scene", fg=54321, sky=5431, images=60, dtype="fp32", step=0,
             clip=False),
        dict(name="adamw8 mlp", op="adamw8", set="mlp", images=400, dtype="fp32", step=1500, clip=False),
        dict(name="adamw8 scene", op="adamw8", set="scene", fg=1363637, sky=136363, images=16, dtype="fp32", step=1500,
             clip=False),
        dict(name="adamw8 ragged bf16 clip", op="adamw8", set="ragged", count=300, low=64, high=2000000, shapes=1,
             dtype="bf16", step=20, clip=True),
        # the largest scene: 5M Gaussians, clipped
        dict(name="adamw8 scene 5M clip", op="adamw8", set="scene", fg=4545455, sky=454545, images=200, dtype="fp32",
             step=7000, clip=True),
        # clipping in place for another optimizer's step
        dict(name="clip scene", op="clip", set="scene", fg=1363637, sky=136363, images=16, dtype="fp32"),
        dict(name="clip ragged fp16", op="clip", set="ragged", count=120, low=1, high=300000, shapes=2, dtype="fp16"),
        # densification: a tenth of the rows pruned, a twentieth appended with zero moments
        dict(name="rows8 scene", op="rows8", set="scene", fg=1363637, sky=136363, keep=0.9, new=0.05, mixed=False),
        # the same early in training, rows in any order
        dict(name="rows8 small", op="rows8", set="scene", fg=20011, sky=1999, keep=0.7, new=0.4, mixed=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("adamw", "adamw8", "clip", "rows8"))
    if op == "rows8":
        fg = _log(rng, 300, 3000000)
        return dict(op=op, set="scene", fg=fg, sky=_log(rng, 1, max(2, fg // 8)), keep=round(rng.uniform(0.3, 1.0), 3),
                    new=round(rng.uniform(0.0, 0.5), 3), mixed=rng.random() < 0.5)
    kind = rng.choice(("mlp", "scene", "scene", "ragged"))
    case = dict(op=op, set=kind, dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")))
    if kind == "mlp":
        case.update(images=_log(rng, 1, 2000))
    elif kind == "scene":
        fg = _log(rng, 300, 3000000 if op == "adamw8" else 2000000)
        case.update(fg=fg, sky=_log(rng, 1, max(2, fg // 8)), images=_log(rng, 1, 2000))
    else:
        case.update(count=_log(rng, 1, 300), low=_log(rng, 1, 100), high=_log(rng, 1000, 1500000),
                    shapes=rng.randrange(1 << 20))
    if op != "clip":
        case.update(step=rng.choice((0, 1, 9, _log(rng, 10, 30000))), clip=rng.random() < 0.5)
    return case


# ---- what a case holds -----------------------------------------------------------------------

def _tensors(case):
    """[(elements, columns, learning rate)] of the case's tensors."""
    if case["set"] == "mlp":
        return [(n, 1, lr) for n, lr in MLP] + [(case["images"] * 32, 32, 2e-4)]
    if case["set"] == "scene":
        rows = {"fg": case["fg"], "sky": case["sky"], "all": case["fg"] + case["sky"]}
        out = [(rows[w] * c, c, lr) for c, w, lr in GROUPS]
        return out if case["op"] == "rows8" else out + [(1, 1, 1e-4), (case["images"] * 32, 32, 2e-4)] + [
            (n, 1, lr) for n, lr in MLP]
    r = random.Random(case["shapes"])
    return [(_log(r, case["low"], case["high"]), 1, r.choice((1e-4, 3e-4, 1e-3))) for _ in range(case["count"])]


def _blocks(n):
    return -(-n // BLOCK)


def _key(ordinal, step):
    return _mix((_mix((SEED + ordinal * MIX_A) & MASK) + step * MIX_B) & MASK)


def _mix(x):
    """Two rounds of multiplication and shift on 32-bit words (Python integers or an int64 tensor)."""
    x = (x * MIX_A) & MASK
    x = x ^ (x >> 15)
    x = (x * MIX_B) & MASK
    return x ^ (x >> 16)


def _scaled(x):
    """x [blocks, 256] -> (|x| times 448 over the block's largest, the block's scale)."""
    top = x.abs().amax(dim=1, keepdim=True)
    top = torch.where(top > 0, top.clamp_min(LEAST), top)
    inv = torch.where(top > 0, TOP / top, torch.zeros_like(top))
    return (x.abs() * inv).clamp_max(TOP), top * (1.0 / TOP)


def _nearest(x, root=False):
    """x [blocks, 256] in 32 bits -> (e4m3 codes rounded to nearest even, scales)."""
    y, scale = _scaled(x)
    q = y.to(torch.float8_e4m3fn).float()
    if root:  # a value that is there stays there
        q = torch.where((y > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return torch.copysign(q, x).to(torch.float8_e4m3fn), scale


def _random(x, u, root=False):
    """x [blocks, 256] in 32 bits, u in [0, 1) -> (e4m3 codes whose expected value is x / scale, scales)."""
    y, scale = _scaled(x)
    exponent = torch.frexp(y).exponent.clamp_min(-5) - 1
    ulp = torch.ldexp(torch.ones_like(y), exponent - 3)
    q = torch.floor(y / ulp + u) * ulp
    if root:
        q = torch.where((y > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return torch.copysign(q, x).to(torch.float8_e4m3fn), scale


def _value(code, scale):
    return code.view(-1, BLOCK).float() * scale.view(-1, 1)


# ---- inputs ----------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _tensors(case)
    t = [x for x in t if x[0] > 0]
    starts, at = [], 0
    for n, _, _ in t:
        starts.append(at)
        at += _blocks(n) * BLOCK
    inside = torch.zeros(at, dtype=torch.bool, device=dev)
    size = torch.empty(at // BLOCK, 1, device=dev)  # each tensor's gradients have a size of their own
    of = torch.rand(len(t), generator=g, device=dev)
    for i, (n, _, _) in enumerate(t):
        inside[starts[i]:starts[i] + n] = True
        size[starts[i] // BLOCK:starts[i] // BLOCK + _blocks(n)] = of[i]
    size = 10.0 ** (-5.0 + 3.0 * size)
    view = lambda flat: [flat[s:s + n].view(-1, c) if c > 1 else flat[s:s + n]  # noqa: E731
                         for s, (n, c, _) in zip(starts, t)]
    normal = lambda: torch.randn(at // BLOCK, BLOCK, generator=g, device=dev)  # noqa: E731
    uniform = lambda: torch.rand(at // BLOCK, BLOCK, generator=g, device=dev)  # noqa: E731
    mask = inside.view(-1, BLOCK)
    s = {"op": case["op"], "inside": inside}
    # gradients spread over some orders of magnitude; what no view of the step saw has none
    spread = size * torch.exp(1.5 * normal())
    grad = normal() * spread * (uniform() < 0.7) * mask
    if case["op"] in ("adamw", "clip", "adamw8"):
        kind = TYPES[case["dtype"]]
        s["grad"] = (grad * (64.0 if kind == torch.float16 else 1.0)).to(kind).view(-1)
        s["grads"] = view(s["grad"])
        value = normal() * mask
        s["param"] = value.to(kind).view(-1)
        s["params"] = view(s["param"])
    if case["op"] == "clip":
        s["max_norm"] = MAX_NORM
        for p, q in zip(s["params"], s["grads"]):
            p.grad = q
        return s
    if case["op"] != "rows8":
        s["master"] = None if kind == torch.float32 else s["param"].float()
        s["masters"] = None if kind == torch.float32 else view(s["master"])
        s["step"], s["clip"] = case["step"], case["clip"]
        s["lrs"] = [lr for _, _, lr in t]
        s["decay"] = 0.01
        s["number"] = torch.cat([torch.full((_blocks(n),), i) for i, (n, _, _) in enumerate(t)]).to(dev)
        s["first"] = torch.cat([torch.arange(_blocks(n)) * BLOCK for n, _, _ in t]).view(-1, 1).to(dev)
        s["lr_blocks"] = torch.tensor(s["lrs"], dtype=torch.float64, device=dev)[s["number"]].view(-1, 1)
        s["max_norm"] = MAX_NORM
        s["eps"] = 1e-15
    # moments as they are after some steps: rows that were never seen have none
    seen = (uniform() < 0.95) * mask
    if case["op"] != "rows8" and case["step"] == 0:
        seen = torch.zeros_like(seen)
    m, v = 0.3 * normal() * spread * seen, (spread * (0.3 + uniform())) ** 2 * seen
    if case["op"] == "adamw":
        s["m"], s["v"] = m.view(-1), v.view(-1)
        s["ms"], s["vs"] = view(s["m"]), view(s["v"])
        return s
    (mc, ms), (rc, rs) = _nearest(m), _nearest(v.sqrt(), root=True)
    s["m"], s["r"], s["m_scale"], s["r_scale"] = mc.view(-1), rc.view(-1), ms.view(-1), rs.view(-1)
    block = lambda flat: [flat[a // BLOCK:a // BLOCK + _blocks(n)] for a, (n, _, _) in zip(starts, t)]  # noqa: E731
    s["moments"] = list(zip(view(s["m"]), view(s["r"]), block(s["m_scale"]), block(s["r_scale"])))
    if case["op"] == "rows8":
        s["index"] = []
        picks = {}
        for n, c, _ in t:
            rows = n // c
            if rows not in picks:  # the groups of one kind of row are indexed alike
                count = max(1, int(case["keep"] * rows))
                if case["mixed"]:
                    kept = torch.randint(0, rows, (count,), generator=g, device=dev)
                else:
                    kept = torch.randperm(rows, generator=g, device=dev)[:count].sort().values
                fresh = torch.full((int(case["new"] * rows),), -1, dtype=torch.int64, device=dev)
                picks[rows] = torch.cat([kept, fresh])
            s["index"].append(picks[rows])
    return s


# ---- one pass --------------------------------------------------------------------------------

def _optim():
    package = os.path.join(ROOT, "relightable3dgaussians-w_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from gsr import optim
    return optim


def _optimizer(s):
    """The optimizer that a training program makes before its first step and keeps: of the case's tensors, as they
    stand before the pass."""
    moments = zip(s["ms"], s["vs"]) if s["op"] == "adamw" else s["moments"]
    names = (("exp_avg", "exp_avg_sq") if s["op"] == "adamw" else
             ("exp_avg", "exp_avg_root", "exp_avg_scale", "exp_avg_root_scale"))
    for p, g in zip(s["params"], s["grads"]):
        p.grad = g
    opt = _optim().AdamW([{"params": [p], "lr": lr} for p, lr in zip(s["params"], s["lrs"])], betas=BETAS, eps=s["eps"],
                         weight_decay=s["decay"], moment_bits=32 if s["op"] == "adamw" else 8,
                         max_grad_norm=s["max_norm"] if s["clip"] else None, seed=SEED)
    for i, (p, m) in enumerate(zip(s["params"], moments)):
        opt.state[p] = {"step": s["step"] - 1, **dict(zip(names, m))} | (
            {} if s["masters"] is None else {"master": s["masters"][i]})
    return opt


def run(s):
    if s["op"] == "clip":
        return _clip(s)
    if s["op"] == "rows8":
        return _rows(s)
    s["step"] += 1
    if own:
        if "optimizer" not in s:
            s["optimizer"] = _optimizer(s)
        s["optimizer"].step()
        found = s["optimizer"].grad_norm
    else:
        found = _plain_step(s)
    return {k: s[k] for k in ("param", "master", "m", "v", "r", "m_scale", "r_scale") if s.get(k) is not None} | (
        {} if found is None else {"norm": found})


def _norm(grad, max_norm):
    norm = grad.double().square().sum().sqrt()
    return torch.stack([norm, (max_norm / (norm + 1e-6)).clamp_max(1.0)]).float()


def _clip(s):
    if own:
        norm = _optim().clip_grad_norm_(s["params"], s["max_norm"])
    else:
        found = _norm(s["grad"], s["max_norm"])
        s["grad"].copy_(s["grad"].float() * found[1])
        norm = found[0]
    return {"norm": norm, "grad": s["grad"]}


def _plain_step(s):
    dev, step = s["grad"].device, s["step"]
    lr = s["lr_blocks"]
    size = (lr / (1.0 - BETAS[0] ** step)).float()
    keep = (1.0 - lr * s["decay"]).float()
    root = 1.0 / math.sqrt(1.0 - BETAS[1] ** step)
    grad = s["grad"].view(-1, BLOCK).float()
    found = None
    if s["clip"]:
        found = _norm(s["grad"], s["max_norm"])
        grad = grad * found[1]
    p = (s["param"] if s["master"] is None else s["master"]).view(-1, BLOCK)
    if s["op"] == "adamw":
        m, v = s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)
    else:
        m, v = _value(s["m"], s["m_scale"]), _value(s["r"], s["r_scale"]).square()
    m = m + (1.0 - BETAS[0]) * (grad - m)
    v = BETAS[1] * v + (1.0 - BETAS[1]) * (grad * grad)
    rms = v.sqrt()
    p.copy_(p * keep - size * (m / (rms * root + s["eps"])))
    if s["master"] is not None:
        s["param"].copy_(s["master"])
    if s["op"] == "adamw":
        s["m"].copy_(m.view(-1))
        s["v"].copy_(v.view(-1))
        return found
    key = torch.tensor([_key(i, step) for i in range(len(s["grads"]))], device=dev)[s["number"]].view(-1, 1)
    word = _mix((s["first"] + torch.arange(BLOCK, device=dev) + key) & MASK)
    for x, u, c, is_root in ((m, word >> 16, "m", False), (rms, word & 0xFFFF, "r", True)):
        code, scale = _random(x, u.float() / 65536.0, is_root)
        s[c].copy_(code.view(-1))
        s[c + "_scale"].copy_(scale.view(-1))
    return found


def _rows(s):
    if own:
        return [list(m) for m in _optim().moments8_rows(s["moments"], s["index"])]
    out = []
    for (mc, rc, ms, rs), index in zip(s["moments"], s["index"]):
        cols = mc.numel() // mc.shape[0]
        new = []
        for code, scale, root in ((mc, ms, False), (rc, rs, True)):
            n = code.numel()
            x = torch.zeros(_blocks(n) * BLOCK, device=code.device)
            x[:n] = code.reshape(-1).float()
            x = (x.view(-1, BLOCK) * scale.view(-1, 1)).view(-1)[:n].view(-1, cols)
            x = torch.where((index >= 0).view(-1, 1), x[index.clamp_min(0)], 0.0)
            y = torch.zeros(_blocks(x.numel()) * BLOCK, device=code.device)
            y[:x.numel()] = x.view(-1)
            c, sc = _nearest(y.view(-1, BLOCK), root)
            new.append((c.view(-1)[:x.numel()].view(-1, cols) if code.dim() > 1 else c.view(-1)[:x.numel()], sc.view(-1)))
        out.append([new[0][0], new[1][0], new[0][1], new[1][1]])
    return out


# ---- the cost and the values in 64 bits ------------------------------------------------------

def work(case):
    n = sum(x[0] for x in _tensors(case))
    if case["op"] == "rows8":
        moved, rows = 0.0, {"fg": case["fg"], "sky": case["sky"], "all": case["fg"] + case["sky"]}
        for c, w, _ in GROUPS:
            kept, new = rows[w] * case["keep"], int(case["new"] * rows[w])
            moved += kept * c * 2 + (kept + new) * c * 2 + (kept + new) * 8 + (2 * kept + new) * c * 8 / BLOCK
        return {"bytes": moved, "flops": 6.0 * n}
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "clip":
        return {"bytes": 2.0 * size * n, "flops": 3.0 * n}
    state = 16.0 if case["op"] == "adamw" else 4.0 + 16.0 / BLOCK
    return {"bytes": (size + (8 if size == 4 else 10) + state) * n,
            "flops": (16.0 if case["op"] == "adamw" else 30.0) * n}


def _e4m3():
    """Every e4m3 value from 0 to 448."""
    return torch.tensor([k * 2.0 ** -9 for k in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16)
                                                           for m in range(8)][:-1], dtype=torch.float64, device="cuda")


def _exact_code(x, u=None, root=False):
    """The values of x's codes, and the scales: u None is the nearest, ties to the even one."""
    table = _e4m3()
    top = x.abs().max(dim=1, keepdim=True).values
    top = torch.where(top > 0, torch.maximum(top, torch.full_like(top, LEAST)), top)
    scale = top / TOP
    y = torch.where(scale > 0, x.abs() / scale, torch.zeros_like(x)).clamp(max=TOP)
    below = (torch.searchsorted(table, y, right=True) - 1).clamp(0, len(table) - 1)
    above = (below + 1).clamp(max=len(table) - 1)
    low, high = table[below], table[above]
    part = torch.where(high > low, (y - low) / (high - low), torch.zeros_like(y))
    up = part + u >= 1.0 if u is not None else (part > 0.5) | ((part == 0.5) & (below % 2 == 1))
    q = torch.where(up, high, low)
    if root:
        q = torch.where(y > 0, q.clamp(min=2.0 ** -9), q)
    return q * torch.sign(x), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        grad = s["grad"].double()
        norm = torch.linalg.vector_norm(grad)
        return {"norm": norm, "grad": grad * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}
    if case["op"] == "rows8":
        out = []
        for (mc, rc, ms, rs), index in zip(s["moments"], s["index"]):
            cols = mc.numel() // mc.shape[0]
            element = (index.view(-1, 1) * cols + torch.arange(cols, device=index.device)).view(-1)
            got = []
            for code, scale, root in ((mc, ms, False), (rc, rs, True)):
                at = element.clamp(min=0)
                x = code.reshape(-1).double()[at] * scale.double()[at // BLOCK] * (element >= 0)
                x = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
                q, sc = _exact_code(x, root=root)
                got.append((q.view(-1)[:element.numel()], sc.view(-1)))
            out.append([got[0][0], got[1][0], got[0][1], got[1][1]])
        return out
    t = [x for x in _tensors(case) if x[0] > 0]
    step = case["step"] + 1
    scale, found = 1.0, None
    if case["clip"]:
        norm = float(torch.linalg.vector_norm(s["grad"].double()))
        scale = min(1.0, s["max_norm"] / (norm + 1e-6))
        found = torch.tensor([norm, scale], dtype=torch.float64)
    out = {k: torch.zeros(s["grad"].numel(), dtype=torch.float64, device="cuda") for k in ("param", "m")}
    if case["op"] == "adamw":
        out["v"] = torch.zeros_like(out["m"])
    else:
        out["r"] = torch.zeros_like(out["m"])
        out["m_scale"] = torch.zeros(s["m_scale"].numel(), dtype=torch.float64, device="cuda")
        out["r_scale"] = torch.zeros_like(out["m_scale"])
    b1, b2 = BETAS
    at = 0
    for k, (n, _, lr) in enumerate(t):
        end = at + _blocks(n) * BLOCK
        g = s["grad"][at:end].double() * scale
        p = (s["param"] if s["master"] is None else s["master"])[at:end].double()
        if case["op"] == "adamw":
            m, v = s["m"][at:end].double(), s["v"][at:end].double()
        else:
            of = slice(at // BLOCK, end // BLOCK)
            m = s["m"][at:end].double() * s["m_scale"][of].double().repeat_interleave(BLOCK)
            v = (s["r"][at:end].double() * s["r_scale"][of].double().repeat_interleave(BLOCK)) ** 2
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g ** 2
        p = p * (1 - lr * s["decay"])
        p = p - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)) ** 0.5 + s["eps"])
        out["param"][at:end] = p
        if case["op"] == "adamw":
            out["m"][at:end], out["v"][at:end] = m, v
        else:
            word = torch.arange(end - at, device="cuda")
            for number in (_exact_key(k, step),):
                word = (word + number) % 2 ** 32
            word = word * 2654435761 % 2 ** 32
            word = word ^ word // 2 ** 15
            word = word * 3037000499 % 2 ** 32
            word = word ^ word // 2 ** 16
            for name, x, u, root in (("m", m, word // 65536, False), ("r", v ** 0.5, word % 65536, True)):
                q, sc = _exact_code(x.view(-1, BLOCK), u.view(-1, BLOCK).double() / 65536, root)
                out[name][at:end] = q.view(-1)
                out[name + "_scale"][of] = sc.view(-1)
        at = end
    if s["master"] is not None:
        out["master"] = out["param"]
    if found is not None:
        out["norm"] = found
    return out


def _exact_key(tensor, step):
    word = (SEED + tensor * 2654435761) % 2 ** 32
    for add in (None, step * 3037000499):
        word = (word + (add or 0)) % 2 ** 32
        word = word * 2654435761 % 2 ** 32
        word ^= word // 2 ** 15
        word = word * 3037000499 % 2 ** 32
        word ^= word // 2 ** 16
    return word
