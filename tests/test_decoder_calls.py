"""What the decoder operators hand to the library, recorded on the CPU: a recorder stands in for the library's entries,
CPU tensors for those on a GPU.  Nothing is computed."""
import types

import pytest
import torch

from d3gs_research_b200 import _lib, group_norm
from d3gs_research_b200.group_norm import _GroupNormAct


class Recorder:
    """Takes the calls of the library: (entry, descriptor's fields where there is one, the other arguments)."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            fields = None
            if hasattr(args[0], "_obj"):   # C.byref(descriptor)
                fields = types.SimpleNamespace(**{k: getattr(args[0]._obj, k) for k, _ in args[0]._obj._fields_})
            self.calls.append((name, fields, args))
            return 256 if name.endswith("workspace_bytes") else 0
        return entry

    def last(self, name):
        return next((f, a) for n, f, a in reversed(self.calls) if n == name)


@pytest.fixture
def recorder(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(_lib, "load", lambda: rec)
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)   # the index of a CPU tensor's device
    return rec


def reaches(at, image, pixel, d):
    """One past the last value that the library reads of a tensor with these strides."""
    return at + 4 * ((d.batch - 1) * image + (d.pixels - 1) * pixel + d.channels)


def extent(t):
    return t.data_ptr() + 4 * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def hooked(x, w, b, unpack):
    """A backward whose saved tensors come back as ``unpack`` makes them, and those of the type's input shape."""
    back = []

    def keep(t):
        back.append(unpack(t))
        return back[-1]

    leaves = [x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, keep):
        y = _GroupNormAct.apply(*leaves, (4, 1e-5, 1))
    torch.autograd.grad(y, leaves, torch.ones_like(y))
    return back


def spread(t):
    """The same values, every second of a wider tensor."""
    wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype)
    wide[..., ::2] = t
    return wide[..., ::2]


def padded(t):
    """The same values with room behind every pixel's channels."""
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, dtype=t.dtype)
    wide[..., 4:4 + t.shape[-1]] = t
    return wide[..., 4:4 + t.shape[-1]]


@pytest.mark.parametrize("view", [lambda t: t[..., 8:48], lambda t: t[:, :, ::2, :40], lambda t: t[:1, :, :, :40].expand(2, -1, -1, -1),
                                  lambda t: t[..., :40].contiguous()])
@pytest.mark.parametrize("unpack", [lambda t: t.clone(memory_format=torch.contiguous_format), padded, spread])
def test_saved_tensors_that_come_back_with_other_strides(recorder, view, unpack):
    """Saved-tensor hooks (``save_on_cpu`` among them) may return a copy laid out anew: the library gets the strides of
    the tensor whose pointer it gets, and reads nothing behind its end."""
    x = view(torch.arange(2 * 6 * 8 * 56, dtype=torch.float32).reshape(2, 6, 8, 56))
    back = hooked(x, torch.ones(40), torch.zeros(40), unpack)
    d, args = recorder.last("d3gs_group_norm_backward")
    x_at, weight_at, bias_at, stats_at = args[1:5]
    got = next(t for t in back if t.shape == x.shape)
    if got.stride(-1) == 1:
        assert x_at == got.data_ptr()
        assert (d.x_batch_stride, d.x_pixel_stride) == group_norm._pixel_strides(got)
        assert reaches(x_at, d.x_batch_stride, d.x_pixel_stride, d) <= extent(got)
    else:                               # copied first
        assert (d.x_batch_stride, d.x_pixel_stride) == (x[0].numel(), 40)
    for at, t in ((weight_at, back[1]), (bias_at, back[2]), (stats_at, back[3])):
        assert (at == t.data_ptr()) == t.is_contiguous()


@pytest.mark.parametrize("unpack", [lambda t: t.double(), lambda t: t[:1], lambda t: t[..., :3]])
def test_saved_tensors_that_come_back_as_something_else(recorder, unpack):
    """Of another type or size they are refused: the library would read what is not there."""
    x = torch.zeros(2, 6, 8, 40)
    with pytest.raises(RuntimeError, match="group_norm_act: a saved tensor came back"):
        hooked(x, torch.ones(40), torch.zeros(40), lambda t: unpack(t) if t.shape == x.shape else t)
    for size in ((40,), (2, 4, 2)):
        with pytest.raises(RuntimeError, match="group_norm_act: a saved tensor came back"):
            hooked(x, torch.ones(40), torch.zeros(40), lambda t: t.double() if t.shape == size else t)
    assert all(name != "d3gs_group_norm_backward" for name, *_ in recorder.calls)


def on_gpu(monkeypatch):
    """CPU tensors that say they are on a GPU: the calls' own checks of their tensors come after those tested here."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)


def calls():
    from d3gs_research_b200 import group_norm_act, muon_step, orthogonalize

    def step(t):
        muon_step([t], [t.clone()], [t.clone()], lr=0.1)
        return t

    return {"group_norm_act": lambda t: group_norm_act(t, 2), "orthogonalize": lambda t: orthogonalize(t), "muon_step": step}


@pytest.mark.parametrize("name", ["group_norm_act", "orthogonalize", "muon_step"])
@pytest.mark.parametrize("grad", [False, True])
def test_calls_under_a_tracer_are_refused(recorder, monkeypatch, name, grad):
    """The trace would hold the allocation of the result and no kernel."""
    from torch.fx.experimental.proxy_tensor import make_fx
    on_gpu(monkeypatch)
    call, x = calls()[name], torch.ones(4, 6)
    if grad and name == "group_norm_act":
        x.requires_grad_()
    with pytest.raises(RuntimeError, match=f"{name}: cannot be traced"):
        torch.jit.trace(call, x)
    for pre in (False, True):
        with pytest.raises(RuntimeError, match=f"{name}: cannot be traced"):
            make_fx(call, pre_dispatch=pre)(x)
    assert not recorder.calls
    call(x.detach())                       # and no longer once the tracer has gone
    assert recorder.calls


@pytest.mark.parametrize("name", ["group_norm_act", "orthogonalize", "muon_step"])
def test_tangents_are_refused(recorder, monkeypatch, name):
    """Forward-mode differentiation would go on without them."""
    import torch.autograd.forward_ad as forward_ad
    from d3gs_research_b200 import group_norm_act
    on_gpu(monkeypatch)
    x = torch.ones(4, 6)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match=f"{name}: has no forward-mode"):
            calls()[name](forward_ad.make_dual(x, x.clone()))
        for k in range(2):
            weights = [torch.ones(6), torch.ones(6)]
            weights[k] = forward_ad.make_dual(weights[k], torch.ones(6))
            with pytest.raises(RuntimeError, match="group_norm_act: has no forward-mode"):
                group_norm_act(x, 2, *weights)
        assert not recorder.calls
        calls()[name](x)                   # inputs without one go through
    assert recorder.calls


def workspace(shapes, dtype=0):
    import ctypes as C
    lib = _lib.load()
    mats = (_lib.OrthoMatrix * len(shapes))()
    for m, (rows, cols) in zip(mats, shapes):
        m.src, m.dst, m.rows, m.cols, m.src_row_stride = 16, 16, rows, cols, cols
    cfg = _lib.OrthoConfig()
    cfg.dtype, cfg.steps, cfg.eps = dtype, 1, 1e-7
    cfg.coefficients[0][:] = (3.4445, -4.775, 2.0315)
    need = lib.d3gs_orthogonalize_workspace_bytes(mats, len(shapes), C.byref(cfg))
    assert need > 0, _lib.last_error()
    return need


@pytest.mark.parametrize("dtype", [0, 1])
def test_workspace_is_that_of_the_largest_batch(dtype):
    """Matrices that stay in shared memory need none; 32 at a time share launches, and all batches one workspace."""
    tiny, wide = (8, 8), (2048, 2048)
    assert workspace([tiny], dtype) == workspace([tiny] * 10000, dtype) <= 4096
    assert workspace([wide] * 32, dtype) == workspace([wide] * 200, dtype) < 33 * workspace([wide], dtype)
    # the large ones fill a batch of their own whatever their order, the small ones need no more
    mixed = [tiny, wide] * 32
    assert workspace(mixed, dtype) == workspace([wide] * 32, dtype)
    assert workspace([wide, (0, 5), tiny, (100, 700)], dtype) <= workspace([wide, tiny, (100, 700)], dtype)
    assert workspace([(0, 4)]) <= 4096


@pytest.mark.parametrize("name", ["group_norm_act", "orthogonalize", "muon_step"])
def test_the_current_device_is_that_of_the_tensors(recorder, monkeypatch, name):
    """With another device current, all calls of the library are made with the tensors' own, forward and backward."""
    current = [7]

    class on:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *exc):
            current.pop()

    seen = []
    original = Recorder.__getattr__

    def spy(self, entry):
        call = original(self, entry)
        return lambda *args: (seen.append((entry, current[-1])), call(*args))[1]

    on_gpu(monkeypatch)
    monkeypatch.setattr(Recorder, "__getattr__", spy)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[-1])
    monkeypatch.setattr(torch.cuda, "device", on)
    x = torch.ones(4, 6)
    if name == "group_norm_act":
        x.requires_grad_()
        y = calls()[name](x)
        torch.autograd.grad(y, x, torch.ones_like(y))
        assert {entry for entry, _ in seen} >= {"d3gs_group_norm_forward", "d3gs_group_norm_backward"}
    else:
        calls()[name](x)
    assert seen and all(device is None for _, device in seen)   # (a CPU tensor's device has no index)
    assert current == [7]
