"""The decoder operators in the calls around a training step: saved-tensor hooks.  Against the same call without them,
and the formula in 64 bits."""
import pytest
import torch

from d3gs_research_b200 import group_norm_act
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
