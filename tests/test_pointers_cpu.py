"""CPU: what the wrappers hand to the library still exists when it is called.  A contiguous copy that only its
.data_ptr() call held is freed before the launch, and a kernel then reads memory of somebody else's."""
import types
import weakref

import pytest
import torch


class Library:
    """In libgsr's place: every call checks that the tensors whose addresses were asked for are alive."""

    def __init__(self):
        self.taken, self.calls = [], []

    def __getattr__(self, name):
        if name.endswith("_partials"):
            return lambda *a: 4

        def call(*args):
            dead = [shape for shape, ref in self.taken if ref() is None]
            assert not dead, f"{name}: freed before the call: {dead}"
            self.calls.append(name)
            self.taken.clear()  # the next call has addresses of its own
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    from gsr import _lib
    made, data_ptr = Library(), torch.Tensor.data_ptr

    def taken(t):
        made.taken.append((tuple(t.shape), weakref.ref(t)))
        return data_ptr(t)
    monkeypatch.setattr(torch.Tensor, "data_ptr", taken)
    monkeypatch.setattr(_lib, "lib", lambda: made)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(_lib, "require_gpu_tensor", lambda t, name: None)
    return made


def context(*saved, **kw):
    return types.SimpleNamespace(saved_tensors=saved, needs_input_grad=(True,) * 8, **kw)


def spread(*shape):
    """A gradient that is not contiguous."""
    return torch.ones(*shape, 2)[..., 0] if len(shape) > 1 or shape[0] > 1 else torch.ones(1).expand(1)


def test_regularisers_backward(library):
    from gsr import train
    ctx = context(torch.ones(6, 3), torch.ones(2, 6), torch.zeros(6, dtype=torch.bool), torch.ones(6, dtype=torch.int32),
                  P=6, V=1, sink_in=(None, None))
    train._FusedViewRegs.backward(ctx, spread(1, 5))
    ctx = context(torch.ones(2, 5), torch.ones(2, 25, 3), torch.ones(20, 25), consts=(1.0, 1.0, 1.0, 0.02, 1), ns=10,
                  env_shape=(2, 25, 3))
    train._RegsTail.backward(ctx, torch.ones(1).expand(2))
    assert library.calls == ["gsr_view_regularisers_backward", "gsr_view_regularisers_tail_backward"]


def test_sky_positions_backward(library):
    from gsr import train
    train._FusedSkyXYZ.backward(context(torch.ones(5, 2), torch.ones(1)), spread(5, 3))
    assert library.calls == ["gsr_sky_xyz_backward"]


def test_channels_backward(library):
    from diff_gaussian_rasterization import _C
    P, H, W = 5, 4, 4
    e = torch.empty(0)
    radii = torch.ones(P, 2, dtype=torch.int32)[:, 0]
    _C.rasterize_gaussians_channels_backward(
        torch.zeros(4), torch.ones(P, 3), radii, torch.ones(P, 4), 4, torch.ones(P, 3), torch.ones(P, 4), 1.0, e,
        torch.eye(4), torch.eye(4), 1.0, 1.0, spread(4, H, W), torch.zeros(3), e, 0, e, e)
    assert library.calls == ["gsr_backward_channels"]


def test_a_step_of_activations_leaves_nothing_behind(library):
    """The activated tensors, and the buffers that collect their gradients, go when a training iteration lets go of
    them: outputs that their own graph node holds as plain attributes would stay for good."""
    import gc

    from gsr import train
    layout = types.SimpleNamespace(P=6, n_fg=4, n_sky=2, src=None)
    p = {"xyz": (4, 3), "sky_angles": (2, 2), "sky_radius": (1,), "scaling": (6, 3), "rotation": (6, 4), "opacity": (6, 1),
         "albedo": (4, 3), "roughness": (4, 1), "metalness": (4, 1)}
    p = {k: torch.ones(shape, requires_grad=True) for k, shape in p.items()}
    for t in p.values():
        t.grad = torch.zeros_like(t)
    scene = types.SimpleNamespace(layout=layout, sky_center=torch.zeros(3), fp=types.SimpleNamespace(params=p), is_sky=None)
    for backward in (False, True):
        model = train.RelitScene.model_fused(scene)
        kept = [weakref.ref(t) for t in vars(model).values() if t is not None]
        sink = model.get_xyz._gsr_sink[0]
        kept += [weakref.ref(t) for t in sink.buf.values()] + [weakref.ref(sink)]
        del sink
        if backward:
            sum(t.sum() for t in vars(model).values() if t is not None).backward()
        del model
        gc.collect()
        assert [r() is None for r in kept] == [True] * len(kept)
