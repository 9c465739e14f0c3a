"""dx of group_norm_act group by group: images and groups whose gradients differ by many orders of magnitude, each held to
its own size.  (A bound from the largest gradient of the whole tensor says little about a small one beside it.)"""
import pytest
import torch

from d3gs_research_b200 import group_norm_act
from test_gpu_group_norm import BF16, EPS, F16, F32, SEQ, U, make, reference, within

pytestmark = pytest.mark.gpu


def by_group(t, groups):
    """[images, pixels, groups, channels of a group]"""
    return t.reshape(t.shape[0], -1, groups, t.shape[-1] // groups)


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
@pytest.mark.parametrize("shape,groups,dtype", [((3, 9, 11, 16), 4, F32), ((3, 9, 11, 16), 4, BF16), ((2, 97, 83, 40), 5, F32),
                                                ((2, 97, 83, 40), 5, BF16), ((2, 50, 60, 15), 3, F16), ((4, 131, 140, 32), 8, F32)])
def test_every_group_by_its_own_size(cuda_device, shape, groups, dtype, act):
    x, dy, w, b = make(shape, groups, dtype, F32)
    # sizes 1 to 1e-3 across images and 1 to 1e-3 across groups: fp16's steps stay relative down to 6e-5
    scale = torch.logspace(0, -1.5 if dtype == F16 else -3, shape[0], device="cuda").view(-1, 1, 1, 1) \
        * torch.logspace(0, -1.5 if dtype == F16 else -3, groups, device="cuda").repeat_interleave(shape[-1] // groups)
    dy = (dy.float() * scale).to(dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps=EPS, act=act), leaves, dy)
    ry, u, want, size, rw, rb, mw, mb = reference(x, groups, w, b, act, dy)
    rows = by_group(x.double(), groups)
    mean = rows.mean((1, 3), keepdim=True)
    rstd = ((rows - mean).square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    # as in the test of forward and backward, with the largest of a group instead of the largest of all
    amp = ((rows.abs() + mean.abs()) * rstd).amax((1, 3), keepdim=True) + 1
    wmax = by_group(w.abs().double().expand(x.shape), groups).amax((1, 3), keepdim=True).clamp(min=1.0)
    size = by_group(size, groups)
    slack = SEQ * U * size + 64 * U * amp * wmax * size.amax((1, 3), keepdim=True)
    within(by_group(dx, groups), by_group(want, groups), slack, "dx")
    ch = (amp * wmax).amax(0).reshape(groups, 1).expand(groups, shape[-1] // groups).reshape(-1)
    within(dw, rw, (SEQ * U + 64 * U * ch) * mw, "dweight")
    within(db, rb, (SEQ * U + 64 * U * ch) * mb, "dbias")
