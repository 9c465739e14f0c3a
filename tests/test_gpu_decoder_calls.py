"""The decoder operators in the calls around a training step: saved-tensor hooks, tracers, tangents, threads; and
waits that give up.  Against the same call without them, and the formula in 64 bits."""
import threading

import pytest
import torch

from d3gs_research_b200 import group_norm_act, muon_step, orthogonalize
from test_gpu_group_norm import BF16, F32, check, make

pytestmark = pytest.mark.gpu

EPS = 1e-5


def padded(t):
    """The same values with room behind every pixel's channels."""
    wide = torch.full((*t.shape[:-1], t.shape[-1] + 24), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., 4:4 + t.shape[-1]] = t
    return wide[..., 4:4 + t.shape[-1]]


# an image in one CTA, and in several
@pytest.mark.parametrize("h,w", [(13, 10), (83, 60)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_saved_tensors_that_come_back_with_other_strides(cuda_device, dtype, h, w):
    """The backward of an input that was read in place, its saved copy dense or padded: ``check`` holds the gradients to
    the formula.  (The width of the loads, and with it the order of the sums, goes by strides and alignment: other strides
    may give other bits.  A dense copy of a dense input has the same ones and gives the same bits.)"""
    dense = lambda t: t.clone(memory_format=torch.contiguous_format)   # noqa: E731
    wide, wide_dy, gamma, beta = make((2, h, 2 * w, 56), 4, dtype, F32)
    gamma, beta = gamma[:40].contiguous(), beta[:40].contiguous()
    for x, dy in ((wide[:, :, :w, 8:48], wide_dy[:, :, :w, 8:48]), (wide[:, :, ::2, :40], wide_dy[:, :, ::2, :40]),
                  (wide[:, :, :w, 8:48].contiguous(), wide_dy[:, :, :w, 8:48].contiguous())):
        _, want = check(x, dy, gamma, beta, 4, "silu")
        for unpack in (None, dense, padded):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack) if unpack else torch.autograd.graph.save_on_cpu():
                _, got = check(x, dy, gamma, beta, 4, "silu")
            if x.is_contiguous() and unpack is not padded:
                assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tracers_and_tangents_are_refused(cuda_device):
    """Neither sees a kernel: a trace would hold the result's allocation alone, a tangent would be lost."""
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(t):
        muon_step([t], [torch.ones_like(t)], [torch.ones_like(t)], lr=0.1)
        return t

    for call in (lambda t: group_norm_act(t, 2), lambda t: orthogonalize(t), step):
        for grad in (False, True):
            x = torch.randn(3, 5, 8, device="cuda")[0].requires_grad_(grad)
            for trace in (lambda: torch.jit.trace(call, x), lambda: make_fx(call)(x)):
                with pytest.raises(RuntimeError, match="cannot be traced"):
                    trace()
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
        before = torch.randn(5, 8, device="cuda")
        after = call(before.clone())
        assert torch.isfinite(after).all() and not torch.equal(after, before)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n", [(200, 300), (384, 3456), (500, 520), (500, 8200)])
def test_a_wait_that_gives_up_with_copies_in_flight(cuda_device, dtype, m, n):
    """One CTA's first tile never comes while its other copies are on their way, or another CTA of the cluster withholds
    all of its own: the loading threads wait for what they asked for, the call returns, its result is NaN, and the next
    call gives the bits it gave before."""
    from d3gs_research_b200 import _lib
    lib = _lib.load()
    u = torch.randn(m, n, generator=torch.Generator(device="cuda").manual_seed(m), device="cuda").to(dtype)
    want = orthogonalize(u)
    for hold in (-2, -3, 1):
        lib.d3gs_test_hooks(300, hold)
        try:
            got = orthogonalize(u)
            torch.cuda.synchronize()
        finally:
            lib.d3gs_test_hooks(0, -1)
        assert torch.isnan(got).all()
        assert torch.equal(orthogonalize(u), want)


@pytest.mark.parametrize("op", ["group_norm", "group_norm_small", "orthogonalize"])
def test_two_threads_with_different_sizes(cuda_device, op):
    """The same kernel with much and with little shared memory, launched by two threads at once: neither call spoils the
    other's launch, and every result has the bits of a call alone."""
    if op == "orthogonalize":
        inputs = [torch.randn(m, n, device="cuda") for m, n in ((64, 64), (128, 190))]
        call = orthogonalize
    else:
        pixels, widths = (70, (16384, 8192)) if op == "group_norm" else (1, (2048, 1792))
        inputs = [torch.randn(1, pixels, c, device="cuda").requires_grad_() for c in widths]

        def call(x):
            y = group_norm_act(x, 32)
            return torch.cat([y.detach(), *torch.autograd.grad(y, x, torch.ones_like(y))])

    want = [call(x) for x in inputs]
    failures, start = [], threading.Barrier(2)

    def work(x, w):
        try:
            stream = torch.cuda.Stream()
            start.wait()
            with torch.cuda.stream(stream):
                bad = sum((call(x) != w).any() for _ in range(1500)).item()
            if bad:
                failures.append(f"{bad} results differ")
        except Exception as e:   # noqa: BLE001 (a thread's exception is lost otherwise)
            failures.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=a) for a in zip(inputs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_launches_of_two_threads(cuda_device):
    """The library's entry from two threads in tight loops (ctypes lets go of the interpreter lock), one with twice the
    shared memory of the other: no launch fails."""
    import ctypes as C
    from d3gs_research_b200 import _lib
    lib = _lib.load()
    failures = []

    def work(channels):
        x = torch.randn(1, 70, channels, device="cuda")
        y, stats = torch.empty_like(x), torch.empty(64, device="cuda")
        d = _lib.GroupNorm(batch=1, pixels=70, x_batch_stride=70 * channels, x_pixel_stride=channels, channels=channels, groups=32,
                           act=1, eps=EPS)
        n = lib.d3gs_group_norm_workspace_bytes(C.byref(d), 0)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        failed = 0
        for k in range(8000):
            failed += lib.d3gs_group_norm_forward(C.byref(d), x.data_ptr(), None, None, y.data_ptr(), stats.data_ptr(),
                                                  ws.data_ptr(), n, stream.cuda_stream) != 0
            if k % 200 == 0:
                stream.synchronize()
        stream.synchronize()
        if failed:
            failures.append((channels, failed, _lib.last_error()))

    threads = [threading.Thread(target=work, args=(c,)) for c in (16384, 8192)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_under_torch_compile(cuda_device):
    """The compiler does not see into the calls and leaves them as they are, with their gradients."""
    def both(x, u):
        return group_norm_act(x * 2, 4) + 1, orthogonalize(u + 0) * 2

    x = torch.randn(2, 9, 11, 40, device="cuda").requires_grad_()
    u = torch.randn(20, 30, device="cuda")
    y, o = both(x, u)
    (dx,) = torch.autograd.grad(y.sum(), x)
    for backend in ("eager", "aot_eager"):
        torch._dynamo.reset()
        z, p = torch.compile(both, backend=backend)(x, u)
        (dz,) = torch.autograd.grad(z.sum(), x)
        assert torch.equal(y, z) and torch.equal(o, p) and torch.equal(dx, dz)
    torch._dynamo.reset()


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_in_the_backward(cuda_device, reentrant):
    """Under activation checkpointing the forward runs again in the backward: the same gradients, to the bit."""
    from torch.utils.checkpoint import checkpoint
    wide, _, gamma, beta = make((2, 31, 29, 56), 4, F32, F32)
    gamma, beta = gamma[:40].contiguous().requires_grad_(), beta[:40].contiguous().requires_grad_()
    wide.requires_grad_()
    layer = lambda t: group_norm_act(group_norm_act(t[..., 8:48], 4, gamma, beta) * 2, 8)   # noqa: E731
    want = torch.autograd.grad(layer(wide).square().sum(), (wide, gamma, beta))
    for t in (wide, gamma, beta):
        t.grad = None
    checkpoint(layer, wide, use_reentrant=reentrant).square().sum().backward()
    assert all(torch.equal(t.grad, w) for t, w in zip((wide, gamma, beta), want))
