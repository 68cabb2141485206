"""AdamW over many separate tensors on the HIP kernels (gsr_adamw_step), with moments in 32 or in
8 bits, and what a training step needs beside it: the global gradient norm it is clipped by
(gsr_grad_norm, gsr_grad_scale) and the rows of 8-bit moments that densification keeps and appends
(gsr_moment_rows).

``AdamW`` takes the place of the reference's torch.optim.Adam(l, lr=0.0, eps=1e-15) over one param
group per Gaussian attribute plus the MLP and the embeddings (gaussian_model.py:259-274,
relit3DGW_model.py:139-150).  With ``moment_bits=32`` its state is torch's (``exp_avg``,
``exp_avg_sq`` of the parameter's shape), so the reference's own surgery on it works unchanged
(gaussian_model.py:438-511); with ``moment_bits=8`` use ``AdamW.replace_rows``.  gsr.train.FlatParams
runs the same kernels over its flat buffer.

GPU tensors only: there is no CPU path.
"""
from __future__ import annotations

import collections
import contextlib
import ctypes as C
import math
import operator
from typing import Iterable, List, NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib

BLOCK = 256  # consecutive elements of a tensor that share one scale of an 8-bit moment
CODE = torch.float8_e4m3fn
_IN_ARGUMENTS = 42  # tensors that gsr_adamw_step takes in one launch without a table in memory
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# gsr_adamw_tensor, gsr_grad_tensor, gsr_moment_rows_tensor (include/gsr.h)
STEP_DTYPE = np.dtype([("param", "u8"), ("grad", "u8"), ("master", "u8"), ("m", "u8"), ("v", "u8"), ("ms", "u8"),
                       ("vs", "u8"), ("n", "i8"), ("first", "i8"), ("step", "i8"), ("step_dev", "u8"), ("lr_dev", "u8"),
                       ("lr", "f8"), ("weight_decay", "f8"), ("ordinal", "i4"), ("param_type", "i4"),
                       ("grad_type", "i4"), ("reserved", "i4")])
GRAD_DTYPE = np.dtype([("grad", "u8"), ("n", "i8"), ("type", "i4"), ("reserved", "i4")])
_ROWS_DTYPE = np.dtype([("src_m", "u8"), ("src_r", "u8"), ("src_ms", "u8"), ("src_rs", "u8"), ("index", "u8"),
                        ("m", "u8"), ("r", "u8"), ("ms", "u8"), ("rs", "u8"), ("src_rows", "i8"), ("rows", "i8"),
                        ("cols", "i4"), ("reserved", "i4")])

_data_ptr = torch.Tensor.data_ptr
_contiguous = torch.Tensor.is_contiguous
_dtype = operator.attrgetter("dtype")
_index = torch.Tensor.get_device


def blocks(n: int) -> int:
    return -(-int(n) // BLOCK)


_STAY = contextlib.nullcontext()


def _on(device: torch.device):
    """The context that makes ``device`` the current one, where it is not."""
    return _STAY if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    """_lib.stream_of for the current device's stream, without the stream object (2 us)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _capturing(device: torch.device) -> bool:
    with _on(device):
        return torch.cuda.is_current_stream_capturing()


def _strided(t: torch.Tensor, name: str) -> None:
    _lib.require_gpu_tensor(t, name)
    if t.layout is not torch.strided:
        raise ValueError(f"{name} must be a dense tensor, got {t.layout}")


# ---- 8-bit moments ------------------------------------------------------------------------

class Moments8(NamedTuple):
    """Adam's two moments of one parameter in 8 bits: ``exp_avg`` and ``exp_avg_root`` (the square
    root of exp_avg_sq) are e4m3 codes of the parameter's shape; element i stands for code *
    scale[i // 256] of its flattened order."""
    exp_avg: torch.Tensor
    exp_avg_root: torch.Tensor
    exp_avg_scale: torch.Tensor
    exp_avg_root_scale: torch.Tensor


_KINDS = [CODE, CODE, torch.float32, torch.float32]


def moments8_empty(shape, device) -> Moments8:
    n = blocks(math.prod(shape))
    return Moments8(torch.empty(shape, dtype=CODE, device=device), torch.empty(shape, dtype=CODE, device=device),
                    torch.empty(n, device=device), torch.empty(n, device=device))


def moments8_zeros(shape, device) -> Moments8:
    m = moments8_empty(shape, device)
    m.exp_avg.view(torch.uint8).zero_()
    m.exp_avg_root.view(torch.uint8).zero_()
    m.exp_avg_scale.zero_()
    m.exp_avg_root_scale.zero_()
    return m


def _check_moments8(m: Sequence[torch.Tensor], name: str, n: Optional[int] = None) -> Moments8:
    if len(m) != 4:
        raise ValueError(f"{name}: 8-bit moments are (exp_avg, exp_avg_root, exp_avg_scale, exp_avg_root_scale)")
    a, r, a_scale, r_scale = m = Moments8(*m)
    device = a.get_device()
    if device < 0 or set(map(_index, m)) != {device} or not _dense(m):
        for t, what in zip(m, m._fields):
            _strided(t, f"{name}.{what}")
            if not t.is_contiguous():
                raise ValueError(f"{name}.{what} must be contiguous")
        raise ValueError(f"{name}: the moments are on different devices")
    if list(map(_dtype, m)) != _KINDS:
        raise TypeError(f"{name}: codes are {CODE} and scales float32, got {list(map(_dtype, m))}")
    n = a.numel() if n is None else n
    if a.numel() != n or r.shape != a.shape:
        raise ValueError(f"{name}: {n} codes of each moment expected, got {tuple(a.shape)} and {tuple(r.shape)}")
    if a_scale.numel() != blocks(n) or r_scale.numel() != blocks(n):
        raise ValueError(f"{name}: {n} elements have {blocks(n)} scales of each moment, got {a_scale.numel()} and "
                         f"{r_scale.numel()}")
    return m


def moments8_encode(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor) -> Moments8:
    """32-bit moments in 8 bits, each code the nearest (a square root above 0 keeps at least the
    least code: m / sqrt(v) stays bounded).  What is not finite becomes NaN; the other elements of
    its block are held as without it."""
    for t, name in ((exp_avg, "exp_avg"), (exp_avg_sq, "exp_avg_sq")):
        _strided(t, name)
        if t.dtype != torch.float32:
            raise TypeError(f"moments8_encode: {name} must be float32, got {t.dtype}")
    if exp_avg.shape != exp_avg_sq.shape or exp_avg.device != exp_avg_sq.device:
        raise ValueError("moments8_encode: the moments differ in shape or device")
    m = moments8_empty(exp_avg.shape, exp_avg.device)
    a, b = _solid(exp_avg.detach()), _solid(exp_avg_sq.detach())
    with _on(a.device):
        _lib.check(_lib.lib().gsr_moments_encode(a.numel(), a.data_ptr(), b.data_ptr(), *map(_data_ptr, m),
                                                 _stream(a.device)), "gsr_moments_encode")
    return m


def moments8_decode(moments: Sequence[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(exp_avg, exp_avg_sq) in 32 bits of 8-bit moments (infinity where a root's square is beyond
    them, from 2^64 on)."""
    m = _check_moments8(moments, "moments")
    a, b = (torch.empty(m.exp_avg.shape, device=m.exp_avg.device) for _ in range(2))
    with _on(a.device):
        _lib.check(_lib.lib().gsr_moments_decode(a.numel(), *map(_data_ptr, m), a.data_ptr(), b.data_ptr(),
                                                 _stream(a.device)), "gsr_moments_decode")
    return a, b


def moments8_rows(moments: Sequence[Sequence[torch.Tensor]], index: Sequence[torch.Tensor]) -> List[Moments8]:
    """Rows of 8-bit moments (the first dimension's), for all parameters at once: row j of the k-th
    result is row index[k][j] of moments[k], or zeros where index[k][j] is -1 (or any other number
    that is not one of the rows): a parameter's rows after pruning and appending
    (gaussian_model.py:438-511).  A row may be taken more than once.  Blocks are those of the new
    rows; codes are rounded to the nearest."""
    if len(moments) != len(index):
        raise ValueError(f"moments8_rows: {len(moments)} moments and {len(index)} indices")
    if not len(moments):
        return []
    desc = np.zeros(len(moments), _ROWS_DTYPE)
    at = desc.ctypes.data
    tensors = [t for m, ix in zip(moments, index) for t in (*m, ix)]
    new = _lib.tensors().gsr_tensors_moment_rows(tensors, at) if len(tensors) == 5 * len(moments) else None
    if new is None:
        _refuse_rows(moments, index)
    device = new[0].device
    with _on(device):
        _lib.check(_lib.lib().gsr_moment_rows(len(moments), at, _stream(device)), "gsr_moment_rows")
    return [Moments8(*new[k:k + 4]) for k in range(0, len(new), 4)]


def _refuse_rows(moments, index) -> None:
    """Says what moments8_rows cannot take of these."""
    device = None
    for k, (m, ix) in enumerate(zip(moments, index)):
        m = _check_moments8(m, f"moments[{k}]")
        _lib.require_gpu_tensor(ix, f"index[{k}]")
        device = m.exp_avg.device if device is None else device
        if m.exp_avg.device != device or ix.device != device:
            raise ValueError("moments8_rows: all moments and indices must be on one device")
        if ix.dtype != torch.int64 or ix.dim() != 1 or not ix.is_contiguous():
            raise ValueError(f"index[{k}] must be a contiguous int64 vector, got {ix.dtype} {tuple(ix.shape)}")
        if m.exp_avg.dim() == 0:
            raise ValueError(f"moments[{k}] has no rows")
    raise ValueError("moments8_rows: moments or indices cannot be used")


# ---- the global gradient norm -------------------------------------------------------------

def _dense(ts: Sequence[torch.Tensor]) -> bool:
    """Whether all tensors are contiguous (a sparse one has no answer to that)."""
    try:
        return all(map(_contiguous, ts))
    except RuntimeError:
        return False


def _solid(g: torch.Tensor) -> torch.Tensor:
    """g, or a copy whose memory holds its values in their order."""
    return g.resolve_neg().contiguous()


def _grads(grads: Iterable[torch.Tensor], what: str) -> Tuple[List[torch.Tensor], np.ndarray, Optional[torch.device]]:
    """(the gradients, dense: the list itself if all are; their table; their device)"""
    grads = grads if isinstance(grads, list) else list(grads)
    desc = np.zeros(len(grads), GRAD_DTYPE)
    if not grads:
        return grads, desc, None
    if _lib.tensors().gsr_tensors_grad_table(grads, desc.ctypes.data) < 0:
        for k, g in enumerate(grads):
            _strided(g, f"{what}: gradient {k}")
            if g.dtype not in _TYPES:
                raise TypeError(f"{what}: gradient {k} is {g.dtype}: float32, bfloat16 and float16 are supported")
            if g.device != grads[0].device:
                raise ValueError(f"{what}: the gradients are on different devices")
        grads = [_solid(g) for g in grads]
        if _lib.tensors().gsr_tensors_grad_table(grads, desc.ctypes.data) < 0:
            raise ValueError(f"{what}: a gradient cannot be made dense")
    return grads, desc, grads[0].device


def _norm(desc: np.ndarray, device: torch.device, max_norm: float, grad_scale: float = 1.0) -> torch.Tensor:
    """gsr_grad_norm over a table of gradients; the current device is ``device``."""
    L = _lib.lib()
    at = desc.ctypes.data
    out = torch.empty(2, device=device)
    work = torch.empty(L.gsr_grad_norm_workspace_bytes(len(desc), at), dtype=torch.uint8, device=device)
    _lib.check(L.gsr_grad_norm(len(desc), at, float(grad_scale), float(max_norm), out.data_ptr(), work.data_ptr(),
                               _stream(device)), "gsr_grad_norm")
    return out


def grad_norm(grads: Iterable[torch.Tensor], max_norm: float = math.inf, grad_scale: float = 1.0) -> torch.Tensor:
    """[norm, coefficient] on the device: the 2-norm of all gradients together, times grad_scale, and
    min(1, max_norm / (norm + 1e-6)), what clipping to max_norm multiplies them by.  Sums in 64 bits
    in a fixed order; no host synchronisation."""
    if not max_norm >= 0:
        raise ValueError(f"grad_norm: max_norm must not be negative, got {max_norm}")
    kept, desc, device = _grads(grads, "grad_norm")
    if device is None:
        raise ValueError("grad_norm: no gradients")
    with _on(device):
        return _norm(desc, device, max_norm, grad_scale)


def clip_grad_norm_(parameters, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ for the 2-norm: scales the parameters' gradients in place so
    that their joint norm is at most max_norm, and returns the norm (a device scalar).  A norm that
    is not finite makes the gradients what torch's multiplication makes them, or raises
    (error_if_nonfinite, which waits for the GPU)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm_: max_norm must not be negative, got {max_norm}")
    grads = _lib.tensors().gsr_tensors_grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    kept, desc, device = _grads(grads, "clip_grad_norm_")
    at = () if kept is grads else [g.data_ptr() for g in grads if g.numel()]  # kept has copies
    if _lib.tensors().gsr_tensors_overlap(desc.ctypes.data, len(desc)) or len(set(at)) != len(at):
        raise ValueError("clip_grad_norm_: a gradient is listed twice, or two share memory")
    if kept is not grads:
        for g, k in zip(grads, kept):
            if k is not g and any(st == 0 and n > 1 for st, n in zip(g.stride(), g.shape)):
                raise ValueError("clip_grad_norm_: an expanded gradient cannot be scaled in place")
    with _on(device):
        out = _norm(desc, device, max_norm)
        if error_if_nonfinite and not math.isfinite(float(out[0])):
            raise RuntimeError("clip_grad_norm_: the gradients' norm is not finite")
        _lib.check(_lib.lib().gsr_grad_scale(len(desc), desc.ctypes.data, out.data_ptr(), _stream(device)),
                   "gsr_grad_scale")
        if kept is grads:
            torch.autograd.graph.increment_version(grads)
        else:
            for g, k in zip(grads, kept):
                if k is g:
                    torch.autograd.graph.increment_version(g)
                else:
                    g.copy_(k)
    return out[0]


# ---- the optimizer ------------------------------------------------------------------------

def _names(moment_bits: int) -> Tuple[str, ...]:
    """What a step looks at in a state, in gsr_tensors_plan's order."""
    return (Moments8._fields if moment_bits == 8 else ("exp_avg", "exp_avg_sq")) + ("master", "step")


class _Plan:
    """The table of one launch list (parameters of one device with one pair of betas and one eps),
    made once and used as long as the optimizer's tensors are those that it was made of (_Seen)."""

    def __init__(self, opt: "AdamW", device, betas, eps, members):
        self.device, self.betas, self.eps, self.bits = device, betas, eps, opt.moment_bits
        self.places = [i for i, _, _ in members]  # among all the optimizer's parameters
        self.groups = [g for _, g, _ in members]
        self.params = [p for _, _, p in members]
        self.states = [opt.state[p] for p in self.params]
        desc = self.desc = np.zeros(len(members), STEP_DTYPE)
        self.at = desc.ctypes.data
        places = self.places_table = np.array(self.places, np.int32)
        self.halves = any(p.dtype != torch.float32 for p in self.params)

        def planned() -> bool:
            return not _lib.tensors().gsr_tensors_plan(self.params, self.states, _names(self.bits), self.bits, opt.capturable,
                                                       device.index, places.ctypes.data, self.at)
        if not planned():
            for p, st in zip(self.params, self.states):
                opt._check_state(p, st)  # says what is wrong, or mends it
            if not planned():
                raise ValueError("AdamW: a state cannot be used")
        self.steps = None
        if not opt.capturable:  # one vector of counts; each state's step is an element of it
            steps = torch.tensor([int(st["step"]) for st in self.states], dtype=torch.int64)
            for st, t in zip(self.states, steps.unbind()):
                st["step"] = t
            self.steps = steps.numpy()
        # a long list's table in device memory, the stream that it is used on, and what it holds
        self.kept, self.kept_on, self.image = None, None, np.zeros(1 + 2 * len(members), np.int64)

    def kept_list(self, stream: int) -> Optional[int]:
        """Device memory for a long list's table, of one stream; none inside a capture, whose graph
        must not go by what later steps write there."""
        n = _lib.lib().gsr_adamw_kept_bytes(len(self.desc))
        if not n or torch.cuda.is_current_stream_capturing():
            return None
        if self.kept is None or self.kept_on != stream:
            self.kept = torch.empty(n, dtype=torch.uint8, device=self.device)
            self.kept_on = stream
            self.image[:] = 0
        return self.kept.data_ptr()

    def grad_table(self) -> np.ndarray:
        out = np.zeros(len(self.desc), GRAD_DTYPE)
        out["grad"], out["n"], out["type"] = self.desc["grad"], self.desc["n"], self.desc["grad_type"]
        return out

    def dense_grads(self, grads: List[torch.Tensor]) -> List[torch.Tensor]:
        """This step's gradients as the kernels take them (kept until the launch), or what is wrong."""
        out = []
        for g, p in zip(grads, self.params):
            if g.layout is not torch.strided:
                raise ValueError(f"AdamW: gradients must be dense tensors, got {g.layout}")
            if g.dtype not in _TYPES:
                raise TypeError(f"AdamW: a gradient is {g.dtype}: float32, bfloat16 and float16 are supported")
            if g.device != p.device or g.numel() != p.numel():
                raise ValueError("AdamW: a gradient differs from its parameter in size or device")
            out.append(_solid(g))
        self.desc["grad_type"] = [_TYPES[g.dtype] for g in out]
        return out


class _Seen:
    """The optimizer's tensors that the plans were made of, as gsr_tensors_current compares them."""

    def __init__(self, opt: "AdamW", params: List[torch.Tensor], grads: List[Optional[torch.Tensor]], left=None):
        """left: what AdamW._left_behind says."""
        T = _lib.tensors()
        self.params, self.keys, self.values = params, list(opt.state), list(opt.state.values())
        self.names = _names(opt.moment_bits)
        words, grad_words = np.zeros((2, len(params), 5), np.int64)
        self.state_words = np.zeros((len(self.values), len(self.names), 5), np.int64)
        if (T.gsr_tensors_describe(params, words.ctypes.data) or T.gsr_tensors_describe(grads, grad_words.ctypes.data) or
                T.gsr_tensors_describe_states(self.values, self.names, self.state_words.ctypes.data)):
            raise TypeError("AdamW: a state is not a dict")
        there = grad_words[:, 2] != -2
        self.words = np.concatenate([words, there[:, None].astype(np.int64), grad_words[:, 2:3]], 1)
        self.at = np.zeros(len(params), np.int64)  # the gradients' addresses
        self.plain = C.c_int(0)
        # the versions of 16-bit parameters when their masters were last theirs; -1: not known, -2: another tensor's
        self.versions = np.full(len(params), -1, np.int64)
        for i, p in enumerate(params if left else ()):
            if p in left:
                self.versions[i] = left[p][1] if left[p][0] == words[i, 0] else -2
        self.written = C.c_int(0)
        self.rest = (self.names, self.state_words.ctypes.data, self.at.ctypes.data, C.byref(self.plain),
                     self.versions.ctypes.data, C.byref(self.written))
        self.words_at = self.words.ctypes.data

    def grads(self, opt: "AdamW") -> Optional[List[Optional[torch.Tensor]]]:
        """The parameters' gradients, if all else is as it was."""
        return _lib.tensors().gsr_tensors_current(opt.param_groups, self.params, self.words_at, opt.state, self.keys,
                                                  self.values, *self.rest)


_RATES = operator.itemgetter("betas", "eps", "lr", "weight_decay")


def _same_constants(a, b) -> bool:
    """Whether the groups' betas and eps (which decide what is launched together) are the same."""
    return len(a) == len(b) and all(x[0] == y[0] and x[1] == y[1] for x, y in zip(a, b))


class _Loaded:
    """A state on its way through torch's load_state_dict, which would cast a dict's tensors to their parameter's
    type."""

    def __init__(self, state: dict):
        self.state = state


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (no amsgrad) over all parameters in a few launches.

    * Parameters: float32, bfloat16 or float16, contiguous, on GPUs; gradients in any of the three.
      A 16-bit parameter has a 32-bit ``master`` in its state, which takes the update; the parameter
      becomes its rounding.  Where the program writes the parameter (a loaded model, a clamp), the next
      step goes on from what it wrote; masters_from_parameters() says which writes cannot be seen.
    * ``moment_bits`` 32: the state is ``step``, ``exp_avg``, ``exp_avg_sq`` as torch's.  8:
      ``exp_avg`` and ``exp_avg_root`` (sqrt of exp_avg_sq) are e4m3 codes with a float scale for
      each 256 elements (``exp_avg_scale``, ``exp_avg_root_scale``): 2 bytes of state per element
      instead of 8.  Codes are rounded up or down at random with this step's exp_avg or root as the
      expected value; ``seed`` and the step, the parameter's place and the element decide, so runs and
      ranks with the same seed agree.  A price in noise: with betas (0.9, 0.999) and gradients of one
      size the root's deviations settle at 17 %, exp_avg_sq's mean is 5 % too large and an update is 18 %
      off (2-norm); elements far below their block's largest fare worse (44 % where a block's gradients
      spread as exp(3 N), 69 % at exp(4 N)): roots below 2^-18 of the largest are held as that.
    * ``max_grad_norm``: gradients are clipped to that joint 2-norm on the way (they are not
      changed); ``grad_norm`` then holds [norm, coefficient] of the last step on the device.  When
      the norm is not finite the step changes neither parameters nor moments; a step count on the
      host still goes up, one on the device (``capturable``) does not.
    * ``capturable``: the step counts are on the device, so step() can be captured into a graph and
      replayed; an ``lr`` that is to change between replays is a float32 device scalar.  Without it
      step() refuses to be captured.

    ``step(grad_scale=s)`` multiplies the gradients by s first (1 / views after a summed exchange).
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, moment_bits=32,
                 max_grad_norm: Optional[float] = None, capturable=False, seed=0):
        if moment_bits not in (8, 32):
            raise ValueError(f"AdamW: moments are held in 8 or 32 bits, got {moment_bits}")
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError(f"AdamW: max_grad_norm must not be negative, got {max_grad_norm}")
        self._moment_bits, self._capturable, self.seed = int(moment_bits), bool(capturable), int(seed)
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        self.grad_norm: Optional[torch.Tensor] = None
        self._plans: Optional[List[_Plan]] = None
        self._seen: Optional[_Seen] = None
        self._left = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    # fixed: the states and the tables are made for them
    moment_bits = property(operator.attrgetter("_moment_bits"))
    capturable = property(operator.attrgetter("_capturable"))

    def __getstate__(self):
        return {**super().__getstate__(), "_moment_bits": self.moment_bits, "_capturable": self.capturable,
                "seed": self.seed, "max_grad_norm": self.max_grad_norm, "grad_norm": None}

    def __setstate__(self, state):
        if "state" in state:  # what load_state_dict hands over is unwrapped
            state = {**state, "state": collections.defaultdict(dict, {
                p: st.state if isinstance(st, _Loaded) else st for p, st in state["state"].items()})}
        super().__setstate__(state)
        for g in self.param_groups:  # a state of another optimizer may lack some
            for k, v in self.defaults.items():
                g.setdefault(k, v)
        self._plans = self._seen = None
        # loaded or copied masters are their parameters' as they are now
        self._left = {p: (p.data_ptr(), p._version) for p, st in self.state.items() if "master" in st}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        self._plans = None
        group = self.param_groups[-1]
        try:
            self._check_group(group)
            for p in group["params"]:
                self._check_param(p)
        except Exception:
            self.param_groups.pop()
            raise

    def _check_group(self, g) -> None:
        b1, b2 = g["betas"]
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {g['betas']}")
        g["betas"] = (b1, b2)  # a list could change without being another
        if not g["eps"] >= 0.0:
            raise ValueError(f"AdamW: eps must not be negative, got {g['eps']}")
        if not g["weight_decay"] >= 0.0:
            raise ValueError(f"AdamW: weight_decay must not be negative, got {g['weight_decay']}")
        for k in ("amsgrad", "maximize", "differentiable"):
            if g.get(k):
                raise ValueError(f"AdamW: {k} is not supported")
        lr = g["lr"]
        if isinstance(lr, torch.Tensor):
            if not self.capturable:
                raise ValueError("AdamW: an lr on the device needs capturable=True")
            if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda:
                raise ValueError("AdamW: an lr tensor is one float32 on the parameters' device")
        elif not lr >= 0.0:
            raise ValueError(f"AdamW: lr must not be negative, got {lr}")

    @staticmethod
    def _check_param(p) -> None:
        _strided(p, "AdamW: a parameter")
        if p.dtype not in _TYPES:
            raise TypeError(f"AdamW: a parameter is {p.dtype}: float32, bfloat16 and float16 are supported")
        if not p.is_contiguous():
            raise ValueError(f"AdamW: parameters must be contiguous, got strides {p.stride()} of {tuple(p.shape)}")

    def _new_state(self, p) -> dict:
        dev = p.device
        st = {"step": torch.zeros((), dtype=torch.int64, device=dev) if self.capturable else 0}
        if self.moment_bits == 8:
            st.update(moments8_zeros(p.shape, dev)._asdict())
        else:
            st.update(exp_avg=torch.zeros(p.shape, device=dev), exp_avg_sq=torch.zeros(p.shape, device=dev))
        if p.dtype != torch.float32:
            st["master"] = p.detach().float()
            self._left[p] = (p.data_ptr(), p._version)
        return st

    def _left_behind(self) -> dict:
        """Of 16-bit parameters whose masters were once made of them or written to them: the address and version that
        they had then."""
        seen = self._seen
        if seen is not None:
            for k in np.flatnonzero(seen.versions != -1):
                self._left[seen.params[k]] = (int(seen.words[k, 0]) if seen.versions[k] != -2 else -1, int(seen.versions[k]))
            seen.versions[:] = -1
        return self._left

    def _master_from(self, p) -> None:
        with torch.no_grad():
            w = self.state[p]["master"].view(p.shape)
            w.copy_(torch.where(w.to(p.dtype) == p, w, p.float()))

    def masters_from_parameters(self) -> None:
        """Makes the 32-bit masters those of their 16-bit parameters: a master whose rounding is its parameter stays,
        another becomes the parameter's value.  step() does so by itself for parameters that were written since
        the last one (by their version counter or another p.data); call this after writing past the counter
        (p.data.copy_(...), a kernel of another library) or between replays of a captured step()."""
        for p, st in self.state.items():
            if st.get("master") is not None:
                self._master_from(p)

    def _check_state(self, p, st) -> None:
        """Raises what a state lacks of what p's step takes; makes a master that is missing."""
        self._check_param(p)
        n = p.numel()
        if self.moment_bits == 8:
            if "exp_avg_root" not in st:
                raise ValueError("AdamW: a state holds no 8-bit moments: load it with load_state_dict, or put "
                                 "moments8_encode's there")
            used = list(_check_moments8([st[k] for k in Moments8._fields], "AdamW: state", n))
            full = []
        else:
            if "exp_avg_sq" not in st:
                raise ValueError("AdamW: a state holds no 32-bit moments: load it with load_state_dict, or put "
                                 "moments8_decode's there")
            full = [("exp_avg", st["exp_avg"]), ("exp_avg_sq", st["exp_avg_sq"])]
            used = [t for _, t in full]
        if p.dtype != torch.float32:
            if st.get("master") is None:
                if _capturing(p.device):  # every replay would begin with the captured master
                    raise RuntimeError("AdamW: take one step() before the capture: it makes the states")
                st["master"] = p.detach().float()
                self._left[p] = (p.data_ptr(), p._version)
            full.append(("master", st["master"]))
            used.append(st["master"])
        for name, t in full:
            _strided(t, f"AdamW: {name}")
            if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
                raise ValueError(f"AdamW: {name} must be {n} contiguous float32, got {tuple(t.shape)} {t.dtype}")
        if self.capturable:
            step = st["step"]
            if not isinstance(step, torch.Tensor) or step.dtype != torch.int64 or step.numel() != 1:
                raise ValueError("AdamW(capturable=True): a step count is one int64 on the device")
            used.append(step)
        for t in used:
            if t.device != p.device:
                raise ValueError(f"AdamW: a state is on {t.device}, its parameter on {p.device}")

    def _make_plans(self, flat, grads) -> None:
        """Plans of the parameters that have a gradient, and what shows that they are still right."""
        owners = [g for g in self.param_groups for _ in g["params"]]
        lists = {}
        for ordinal, (p, g, grad) in enumerate(zip(flat, owners, grads)):
            if grad is None:
                continue
            if not self.state[p]:
                if _capturing(p.device):  # every replay would begin with zero moments
                    raise RuntimeError("AdamW: take one step() before the capture: it makes the states")
                self.state[p] = self._new_state(p)
            lists.setdefault((p.device, tuple(g["betas"]), float(g["eps"])), []).append((ordinal, g, p))
        self._plans = None  # none, if one of these is refused
        plans = [_Plan(self, *key, members) for key, members in lists.items()]
        every = plans[0].desc if len(plans) == 1 else np.concatenate([plan.desc for plan in plans] or [np.zeros(0, STEP_DTYPE)])
        if _lib.tensors().gsr_tensors_written_overlap(every.ctypes.data, len(every), self.moment_bits):
            raise ValueError("AdamW: parameters or states share memory")
        self._seen = _Seen(self, flat, grads, self._left_behind())
        self._left = {}
        self._rates = None
        self._plans = plans

    def _current(self) -> Tuple[List[_Plan], List[Optional[torch.Tensor]]]:
        """The plans and all parameters' gradients, the plans made anew where a tensor is not what it was."""
        rates = list(map(_RATES, self.param_groups))
        if self._plans is not None and (self._rates is None or _same_constants(rates, self._rates)):
            grads = self._seen.grads(self)
            if grads is not None:
                if self.capturable or rates != self._rates:
                    self._set_rates(rates)
                return self._plans, grads
        flat = [p for g in self.param_groups for p in g["params"]]
        grads = [p.grad for p in flat]
        self._make_plans(flat, grads)
        self._set_rates(rates)
        grads = self._seen.grads(self)
        if grads is None:
            raise RuntimeError("AdamW: parameters or states changed during step()")
        return self._plans, grads

    def _set_rates(self, rates) -> None:
        """Learning rates and weight decays as they are now, into the tables."""
        for g in self.param_groups:
            self._check_group(g)
        for plan in self._plans:
            lrs = [g["lr"] for g in plan.groups]
            if self.capturable:
                on_device = [isinstance(x, torch.Tensor) for x in lrs]
                for x, d in zip(lrs, on_device):
                    if d and x.device != plan.device:
                        raise ValueError(f"AdamW: an lr is on {x.device}, its parameters on {plan.device}")
                plan.desc["lr_dev"] = [x.data_ptr() if d else 0 for x, d in zip(lrs, on_device)]
                lrs = [0.0 if d else x for x, d in zip(lrs, on_device)]
            plan.desc["lr"] = lrs
            plan.desc["weight_decay"] = [g["weight_decay"] for g in plan.groups]
        self._rates = rates

    def step(self, closure=None, *, grad_scale: float = 1.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self.max_grad_norm is not None and not self.max_grad_norm >= 0:
            raise ValueError(f"AdamW: max_grad_norm must not be negative, got {self.max_grad_norm}")
        plans, grads = self._current()
        if not plans:
            return loss
        if self.max_grad_norm is not None and len({p.device for p in plans}) > 1:
            raise ValueError("AdamW: max_grad_norm needs all parameters on one device")
        if not self.capturable and any(_capturing(plan.device) for plan in plans):
            raise RuntimeError("AdamW: a captured step() needs capturable=True (the step count would stay the "
                               "captured one)")
        clip, max_norm = None, -1.0
        seen, held = self._seen, [grads]  # kept until the launches
        if seen.written.value:
            for p, g, version in zip(seen.params, grads, seen.versions):
                if g is not None and version != -1 and p._version != version:
                    self._master_from(p)
        for plan in plans:
            every = len(plan.places) == len(grads)
            if seen.plain.value:
                plan.desc["grad"] = seen.at if every else seen.at[plan.places]
                plan.desc["grad_type"] = seen.words[:, 6] if every else seen.words[plan.places, 6]
            else:  # some are of another type than before, have to be copied, or are refused
                dense = plan.dense_grads(grads if every else [grads[i] for i in plan.places])
                held.append(dense)
                plan.desc["grad"] = list(map(_data_ptr, dense))
                seen.words[plan.places, 6] = plan.desc["grad_type"]
        if self.max_grad_norm is not None:
            device = plans[0].device
            if len(plans) == 1:  # the step finds the norm itself
                clip, max_norm = torch.empty(2, device=device), self.max_grad_norm
            else:
                with _on(device):
                    clip = _norm(np.concatenate([plan.grad_table() for plan in plans]), device, self.max_grad_norm,
                                 grad_scale)
            self.grad_norm = clip
        for plan in plans:
            with _on(plan.device):
                self._launch(plan, clip, max_norm, grad_scale)
        del held
        return loss

    def _launch(self, plan: _Plan, clip, max_norm: float, grad_scale) -> None:
        desc, L, work, stream = plan.desc, _lib.lib(), None, _stream(plan.device)
        kept = plan.kept_list(stream) if len(desc) > _IN_ARGUMENTS else None
        if self.capturable or len(desc) > _IN_ARGUMENTS or max_norm >= 0:
            work = torch.empty(L.gsr_adamw_workspace_bytes(len(desc), plan.at, max_norm >= 0), dtype=torch.uint8,
                               device=plan.device)
        if plan.steps is not None:
            desc["step"] = plan.steps + 1
        _lib.check(L.gsr_adamw_step(len(desc), plan.at, self.moment_bits, plan.betas[0], plan.betas[1], plan.eps,
                                    self.seed & 0xffffffff, float(grad_scale), max_norm,
                                    None if clip is None else clip.data_ptr(), None if work is None else work.data_ptr(),
                                    kept, None if kept is None else plan.image.ctypes.data, stream), "gsr_adamw_step")
        if plan.steps is not None:
            plan.steps += 1
        # the kernel wrote through raw pointers: saved-tensor checks and caches see it
        torch.autograd.graph.increment_version(plan.params)
        if plan.halves and not torch.cuda.is_current_stream_capturing():  # a capture steps nothing yet
            _lib.tensors().gsr_tensors_versions(plan.params, plan.places_table.ctypes.data, self._seen.versions.ctypes.data)

    # ---- states from elsewhere, and rows that come and go

    def load_state_dict(self, state_dict) -> None:
        """Takes this class's or torch.optim.Adam / AdamW's state, with moments in either width (they
        are converted to this optimizer's).  A weight decay is AdamW's, whatever the state is of."""
        last = self.register_load_state_dict_pre_hook(AdamW._before_load)  # behind the program's own: it sees what they return
        try:
            super().load_state_dict(state_dict)
        finally:
            last.remove()

    def _before_load(self, state_dict) -> Optional[dict]:
        """state_dict with its states as this optimizer holds them.  All that can be refused is refused here, before
        anything changes."""
        saved, groups = state_dict["state"], state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            return None  # torch says what is wrong
        for st in saved.values():
            if "max_exp_avg_sq" in st:
                raise ValueError("AdamW: an amsgrad state cannot be loaded")
        ids = [i for g in groups for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for g in groups:
            self._check_group({**self.defaults, **g})
        return {**state_dict, "state": {i: _Loaded(self._converted(p, saved[i])) for i, p in zip(ids, params) if saved.get(i)}}

    def _converted(self, p, saved) -> dict:
        take = lambda t: torch.as_tensor(t).detach().to(p.device).clone()  # noqa: E731
        alike = lambda t: take(t).reshape(p.shape).contiguous()  # noqa: E731
        step = int(saved["step"])
        st = {"step": torch.full((), step, dtype=torch.int64, device=p.device) if self.capturable else step}
        sizes = {k: torch.as_tensor(saved[k]).numel() for k in ("exp_avg", "exp_avg_root", "exp_avg_sq", "master") if k in saved}
        if set(sizes.values()) != {p.numel()}:
            raise ValueError(f"AdamW: a state of {sizes} elements cannot be loaded for {tuple(p.shape)}")
        if "exp_avg_root" in saved:
            if any(k not in saved for k in Moments8._fields):
                raise ValueError(f"AdamW: a state of 8-bit moments has {Moments8._fields}, got {tuple(saved)}")
            m = _check_moments8([alike(saved[k]) for k in Moments8._fields[:2]] +
                                [take(saved[k]).contiguous() for k in Moments8._fields[2:]], "AdamW: state", p.numel())
            if self.moment_bits == 8:
                st.update(m._asdict())
            else:
                st["exp_avg"], st["exp_avg_sq"] = moments8_decode(m)
        else:
            m, v = (alike(saved[k]).float() for k in ("exp_avg", "exp_avg_sq"))
            if self.moment_bits == 8:
                st.update(moments8_encode(m, v)._asdict())
            else:
                st.update(exp_avg=m, exp_avg_sq=v)
        if p.dtype != torch.float32:
            st["master"] = alike(saved["master"]).float() if "master" in saved else p.detach().float()
        return st

    def replace_rows(self, old: Sequence[torch.Tensor], new: Sequence[torch.Tensor],
                     index: Sequence[torch.Tensor]) -> None:
        """Puts new[k] into old[k]'s place, its state's rows taken from old[k]'s: row j has the moments
        of old row index[k][j], or zeros where that is -1 (cat_tensors_to_optimizer and
        _prune_optimizer, gaussian_model.py:438-511, for all groups at once).  The step count stays;
        a 16-bit parameter's kept rows keep their 32-bit master."""
        if not len(old) == len(new) == len(index):
            raise ValueError(f"replace_rows: {len(old)} old and {len(new)} new parameters and {len(index)} indices")
        where = {id(p): (g, k) for g in self.param_groups for k, p in enumerate(g["params"])}
        seen, taken = set(), set()
        others = set(where) - set(map(id, old))
        for p, q, ix in zip(old, new, index):
            if id(p) not in where or id(p) in seen:
                raise ValueError("replace_rows: a parameter is not the optimizer's, or is listed twice")
            if id(q) in taken or id(q) in others:
                raise ValueError("replace_rows: a new parameter is listed twice, or is another one of the optimizer's")
            seen.add(id(p))
            taken.add(id(q))
            self._check_param(q)
            if p.dim() == 0 or q.shape[1:] != p.shape[1:] or q.dtype != p.dtype or q.device != p.device:
                raise ValueError(f"replace_rows: {tuple(q.shape)} {q.dtype} cannot take the place of "
                                 f"{tuple(p.shape)} {p.dtype}")
            if ix.dtype != torch.int64 or ix.dim() != 1 or ix.numel() != q.shape[0] or ix.device != p.device:
                raise ValueError(f"replace_rows: an index is an int64 vector of the {q.shape[0]} new rows on the "
                                 "parameter's device")
        held = [k for k, p in enumerate(old) if self.state.get(p)]
        states = {}
        if self.moment_bits == 8:
            byd = {}
            for k in held:
                byd.setdefault(old[k].device, []).append(k)
            for ks in byd.values():
                rows = moments8_rows([[t.view(old[k].shape) if t.dtype == CODE else t for t in
                                       (self.state[old[k]][f] for f in Moments8._fields)] for k in ks],
                                     [index[k].contiguous() for k in ks])
                for k, m in zip(ks, rows):
                    states[k] = m._asdict()
        for k in held:
            p, st, ix = old[k], self.state[old[k]], index[k]
            there = (ix >= 0) & (ix < p.shape[0])
            at = torch.where(there, ix, 0)
            mask = there.view(-1, *([1] * (p.dim() - 1)))

            def rows(t, other):
                if p.shape[0] == 0:
                    return torch.zeros(new[k].shape, device=p.device) + other
                return torch.where(mask, t.view(p.shape).index_select(0, at), other)
            with torch.no_grad():
                if self.moment_bits == 32:
                    zero = torch.zeros((), device=p.device)
                    states[k] = {"exp_avg": rows(st["exp_avg"], zero), "exp_avg_sq": rows(st["exp_avg_sq"], zero)}
                if "master" in st:
                    states[k]["master"] = rows(st["master"], new[k].detach().float())
            states[k]["step"] = st["step"]
        for p in old:
            self.state.pop(p, None)
        left = self._left_behind()
        for k, (p, q) in enumerate(zip(old, new)):
            g, at = where[id(p)]
            g["params"][at] = q
            left.pop(p, None)
            if k in states:
                self.state[q] = states[k]
                if "master" in states[k]:
                    left[q] = (q.data_ptr(), q._version)
        self._plans = None
