"""The decoder operators in the calls around a training step: saved-tensor hooks, tracers, tangents; and waits that give
up.  Against the same call without them, and the formula in 64 bits."""
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
