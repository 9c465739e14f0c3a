"""group_norm_act against its formula in 64 bits: types, group layouts, odd sizes, strides, empty and single-pixel
images, non-finite values, streams and graphs.

Tolerances.  The kernels compute in 32 bits and round once to the output's type, so an output may be off by half a
step of its type (eps/2 relative) plus the 32-bit arithmetic before it.  That arithmetic is a dozen roundings of
values of size (|x| + |mean|) * rstd * |w| and, for sums, at most SEQ additions in a row of a thread, a warp's tree
or a join: SEQ * 2^-24 of the sum of magnitudes bounds what they lose.
"""
import math

import pytest
import torch
from torch.nn import functional as F

from d3gs_research_b200 import group_norm_act

pytestmark = pytest.mark.gpu

EPS = 1e-5
U = 2.0 ** -24
SEQ = 512
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def reference(x, groups, w, b, act, dy=None):
    """y, and with dy: dx, dw, db and the sums of magnitudes of the last two, in float64."""
    c = x.shape[-1]
    x, w, b = (None if t is None else t.detach().double() for t in (x, w, b))
    rows = x.reshape(x.shape[0], -1, groups, c // groups)
    mean = rows.mean((1, 3), keepdim=True)
    rstd = ((rows - mean).square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    xhat = ((rows - mean) * rstd).reshape(x.shape)
    ww = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w
    u = xhat * ww + (0 if b is None else b)
    y = {"none": lambda v: v, "silu": F.silu, "gelu": F.gelu}[act](u)
    if dy is None:
        return y, u
    if act == "silu":
        s = torch.sigmoid(u)
        slope = s * (1 + u * (1 - s))
    elif act == "gelu":
        slope = 0.5 * (1 + torch.erf(u / math.sqrt(2))) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    else:
        slope = torch.ones_like(u)
    du = dy.double() * slope
    d = (du * ww).reshape(rows.shape)
    xh = xhat.reshape(rows.shape)
    dx = (rstd * (d - d.mean((1, 3), keepdim=True) - xh * (d * xh).mean((1, 3), keepdim=True))).reshape(x.shape)
    flat = (-1, c)
    # what one value of dx is made of: its rounding errors are of this size
    size = (rstd * (d.abs() + d.abs().mean((1, 3), keepdim=True) * (1 + xh.abs()))).reshape(x.shape)
    return y, u, dx, size, (du * xhat).reshape(flat).sum(0), du.reshape(flat).sum(0), \
        (du * xhat).abs().reshape(flat).sum(0), du.abs().reshape(flat).sum(0)


def within(got, ref, slack, what):
    half = torch.finfo(got.dtype).eps / 2
    # the smallest steps of a 16-bit float are absolute (fp16 keeps 2^-25 below its normal range)
    bound = half * ref.abs() * 1.001 + slack + (2.0 ** -25 if got.dtype == F16 else 0.0)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = (err - bound).max().item() if err.numel() else -1.0
    assert worst <= 0, f"{what}: over its bound by {worst} (largest error {err.max().item()})"


def make(shape, groups, dtype, wdtype, seed=0, offset=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g, device="cuda") * (0.5 + torch.rand(c, generator=g, device="cuda"))
         + offset * torch.randn(c, generator=g, device="cuda")).to(dtype)
    dy = torch.randn(shape, generator=g, device="cuda").to(dtype)
    w = b = None
    if wdtype is not None:
        w = (1 + 0.3 * torch.randn(c, generator=g, device="cuda")).to(wdtype)
        b = (0.3 * torch.randn(c, generator=g, device="cuda")).to(wdtype)
    return x, dy, w, b


def check(x, dy, w, b, groups, act, what=""):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps=EPS, act=act)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    ry, u, dx, size, dw, db, mw, mb = reference(x, groups, w, b, act, dy)
    xf = x.double()
    rows = xf.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    mean = rows.mean((1, 3), keepdim=True)
    rstd = ((rows - mean).square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    amp = ((rows.abs() + mean.abs()) * rstd).reshape(x.shape) + 1
    wmax = 1.0 if w is None else max(1.0, w.abs().max().item())
    within(y.detach(), ry, 32 * U * amp * wmax * (1 + u.abs()), f"y {what}")
    # the relative error of a slope is that of u times the curvature (below 1.2) and the statistics' own
    rel = 64 * U * amp.amax() * wmax
    within(got[0], dx, SEQ * U * size + rel * size.amax(), f"dx {what}")
    if w is not None:
        within(got[1], dw, (SEQ * U + rel) * mw + U, f"dweight {what}")
        within(got[2], db, (SEQ * U + rel) * mb + U, f"dbias {what}")
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, groups, w, b, eps=EPS, act=act), y.detach())
    return y.detach(), got


CASES = [
    # shape, groups, type, weight type, act
    ((1, 1, 1, 1), 1, F32, F32, "none"),             # one value: the variance is zero
    ((2, 1, 1, 8), 8, BF16, F32, "silu"),            # one value per group
    ((2, 3, 5), 5, F32, F32, "silu"),                # one spatial axis, a channel per group
    ((3, 6), 2, F16, F16, "gelu"),                   # no spatial axis
    ((1, 7, 9, 9), 3, BF16, BF16, "silu"),           # odd channels, the image ends inside a 16-byte vector
    ((1, 7, 9, 9), 1, F32, None, "gelu"),            # the same in 32 bits, without weights
    ((3, 5, 7, 12), 4, F16, F32, "silu"),            # images start off a 16-byte boundary
    ((3, 5, 7, 5), 1, BF16, F32, "none"),            # images start off every boundary
    ((2, 33, 17, 80), 5, F32, F32, "gelu"),
    ((2, 33, 17, 80), 5, BF16, F32, "silu"),
    ((1, 64, 64, 512), 32, F16, F32, "silu"),
    ((1, 2, 2, 2050), 2, BF16, F32, "silu"),         # more vectors in a pixel than threads
    ((1, 2, 3, 515), 5, F32, F32, "none"),           # the same, odd
    ((2, 2, 2, 16384), 64, F16, F32, "silu"),        # the most channels
    ((2, 200, 301, 32), 8, BF16, F32, "silu"),       # many chunks, a ragged last one
    ((2, 201, 301, 3), 3, F32, F32, "gelu"),         # colour images: instance normalisation
    ((5, 401, 399, 32), 1, F16, F32, "silu"),        # several turns of images
    ((2, 25, 30, 64), 8, F32, F32, "silu"),          # a forward in one launch, a backward in three
    ((3, 20, 40, 80), 5, BF16, BF16, "gelu"),        # one launch for either, parameter gradients in another
    ((1, 3, 2, 2048), 32, BF16, F32, "silu"),        # the most channels that a CTA takes alone
    ((1, 3, 2, 2056), 257, BF16, F32, "silu"),       # and one vector more
    ((150, 31, 33, 64), 8, BF16, F32, "silu"),       # an image for every SM
    ((150, 9, 11, 7), 7, F16, F32, "gelu"),          # the same, odd
]


@pytest.mark.parametrize("shape,groups,dtype,wdtype,act", CASES)
def test_forward_and_backward(cuda_device, shape, groups, dtype, wdtype, act):
    x, dy, w, b = make(shape, groups, dtype, wdtype)
    check(x, dy, w, b, groups, act, str(shape))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_mean_far_from_zero(cuda_device, dtype):
    """A mean of a hundred spreads: what is lost is the rounding of x itself, not the square of the mean."""
    x, dy, w, b = make((2, 90, 91, 16), 4, dtype, F32, offset=0.0)
    x = (x.float() + 100).to(dtype)
    check(x, dy, w, b, 4, "silu")


def test_background_before_the_object(cuda_device):
    """The first half of the image is empty: the rows a thread starts with are far from the mean of the rest."""
    x, dy, w, b = make((1, 128, 200, 32), 8, F32, F32, offset=0.0)
    x += 50
    x[:, :64] = 0
    check(x, dy, w, b, 8, "silu")


@pytest.mark.parametrize("size", [9, 90])
def test_only_weight_or_only_bias(cuda_device, size):
    x, dy, w, b = make((2, size, 11, 24), 3, F32, F32)
    for ww, bb in ((w, None), (None, b)):
        leaf = (ww if ww is not None else bb).detach().requires_grad_()
        y = group_norm_act(x, 3, leaf if ww is not None else None, leaf if bb is not None else None, eps=EPS)
        (g,) = torch.autograd.grad(y, leaf, dy)
        r = reference(x, 3, ww, bb, "silu", dy)
        within(y.detach(), r[0], 1e-5, "y")
        within(g, r[4] if ww is not None else r[5], 1e-5 * (r[6] if ww is not None else r[7]), "gradient")


# a CTA an image, and several
@pytest.mark.parametrize("h,w", [(13, 10), (83, 60)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_inputs(cuda_device, dtype, h, w):
    """A slice of the channels, a view of a channels-first tensor, every other column, one pixel for all."""
    x, dy, gamma, beta = make((2, h, w, 40), 4, dtype, F32)
    base, _ = check(x, dy, gamma, beta, 4, "silu")
    wide = torch.zeros(2, h, w, 56, dtype=dtype, device="cuda")
    wide[..., 8:48] = x
    wide_dy = torch.zeros(2, h, w, 47, dtype=dtype, device="cuda")
    wide_dy[..., 3:43] = dy
    check(wide[..., 8:48], wide_dy[..., 3:43], gamma, beta, 4, "silu")
    check(wide[..., 5:45], dy, gamma, beta, 4, "silu")
    nchw = x.permute(0, 3, 1, 2).contiguous()
    y, _ = check(nchw.permute(0, 2, 3, 1), dy.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1), gamma, beta, 4, "silu")
    assert torch.equal(y, base)
    check(x[:, :, ::2], dy[:, :, ::2], gamma, beta, 4, "silu")
    check(x[:, 1:, 1:], dy[:, 1:, 1:], gamma, beta, 4, "silu")
    check(x, dy[:, :1, :1].expand(x.shape), gamma, beta, 4, "silu")
    check(x[:1].expand(x.shape), dy, gamma, beta, 4, "silu")
    nhwc = torch.empty(2, 40, h, w, device="cuda", dtype=dtype, memory_format=torch.channels_last)
    nhwc.copy_(nchw)
    y, _ = check(nhwc.permute(0, 2, 3, 1), dy, gamma, beta, 4, "silu")
    assert torch.equal(y, base)
    # a scalar loss hands back a gradient without extent
    leaf = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(group_norm_act(leaf, 4, gamma, beta, eps=EPS).sum(), leaf)
    r = reference(x, 4, gamma, beta, "silu", torch.ones_like(x))
    within(dx, r[2], 1e-4 * r[3].amax(), "dx of a sum")


@pytest.mark.parametrize("shape", [(0, 4, 4, 8), (2, 0, 4, 8)])
def test_empty(cuda_device, shape):
    x = torch.empty(shape, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    b = torch.ones(8, device="cuda", requires_grad=True)
    y = group_norm_act(x, 2, w, b)
    assert y.shape == shape
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("width", [30, 300])
def test_non_finite_values_stay_in_their_group(cuda_device, width):
    x, dy, w, b = make((2, 21, width, 16), 4, F32, F32)
    clean = group_norm_act(x, 4, w, b, eps=EPS)
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = x.clone()
        z[1, 11, 7, 5] = bad                     # image 1, group 1
        y = group_norm_act(z, 4, w, b, eps=EPS)
        assert torch.isnan(y[1, ..., 4:8]).all()
        y[1, ..., 4:8] = clean[1, ..., 4:8]
        assert torch.equal(y, clean)


def test_saturated_activation(cuda_device):
    """Weights that drive the activation far into both ends: no NaN from exp overflow."""
    x, dy, w, b = make((1, 20, 20, 8), 2, F32, F32)
    for act in ("silu", "gelu"):
        leaf = x.detach().requires_grad_()
        y = group_norm_act(leaf, 2, w * 1e3, b, eps=EPS, act=act)
        (dx,) = torch.autograd.grad(y, leaf, dy)
        r = reference(x, 2, w * 1e3, b, act, dy)
        assert torch.isfinite(y).all() and torch.isfinite(dx).all()
        within(y.detach(), r[0], 1e-5 * r[0].abs().amax(), act)


def test_gradient_against_differences(cuda_device):
    """The gradient's product with a direction against central differences of the 64-bit formula.  Step 1e-4: the
    third-order term is below 1e-7 of the value, the 64-bit rounding below 1e-10; the kernel's own error decides."""
    x, dy, w, b = make((2, 6, 5, 12), 3, F32, F32)
    g = torch.Generator(device="cuda").manual_seed(3)
    for act in ("none", "silu", "gelu"):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = group_norm_act(leaves[0], 3, leaves[1], leaves[2], eps=EPS, act=act)
        grads = torch.autograd.grad(y, leaves, dy)
        for k in range(3):
            v = torch.randn(leaves[k].shape, generator=g, device="cuda").double()
            ends = []
            for h in (1e-4, -1e-4):
                at = [t.double() for t in (x, w, b)]
                at[k] = at[k] + h * v
                ends.append((reference(at[0], 3, at[1], at[2], act)[0] * dy.double()).sum())
            want = (ends[0] - ends[1]) / 2e-4
            size = (grads[k].double() * v).abs().sum()
            assert abs((grads[k].double() * v).sum() - want) <= 1e-5 * size


def test_same_result_every_time_and_on_another_stream(cuda_device):
    x, dy, w, b = make((3, 150, 170, 32), 8, BF16, F32)
    base = check(x, dy, w, b, 8, "silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = []
        for _ in range(3):
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = group_norm_act(leaves[0], 8, leaves[1], leaves[2], eps=EPS)
            again.append((y.detach(), torch.autograd.grad(y, leaves, dy)))
    torch.cuda.current_stream().wait_stream(side)
    for y, grads in again:
        assert torch.equal(y, base[0])
        assert all(torch.equal(p, q) for p, q in zip(grads, base[1]))


def test_captured_and_replayed(cuda_device):
    """Forward and backward inside one graph, replayed on new inputs; two graphs replayed on two streams at once."""
    made = []
    for seed in (1, 2):
        x, dy, w, b = make((2, 60, 70, 24), 3, BF16, F32, seed=seed)
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]

        def step():
            y = group_norm_act(leaves[0], 3, leaves[1], leaves[2], eps=EPS)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        made.append((graph, leaves, dy, out, step))
    for seed in (11, 12):
        for k, (graph, leaves, dy, out, step) in enumerate(made):
            nx, ndy, nw, nb = make((2, 60, 70, 24), 3, BF16, F32, seed=seed + 100 * k)
            with torch.no_grad():
                for t, n in zip((*leaves, dy), (nx, nw, nb, ndy)):
                    t.copy_(n)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in made]
        for s, (graph, *_) in zip(streams, made):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for graph, leaves, dy, out, step in made:
            assert all(torch.equal(p, q) for p, q in zip(out, step()))


@pytest.mark.parametrize("size", [4, 64])
def test_first_gradients_of_a_graph_that_is_kept(cuda_device, size):
    """create_graph gives the same gradients; a second derivative is refused, not wrong."""
    x, dy, w, b = make((2, size, size, 8), 2, F32, F32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = group_norm_act(leaves[0], 2, leaves[1], leaves[2])
    plain = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    kept = torch.autograd.grad(y, leaves, dy, create_graph=True)
    assert all(torch.equal(p, k) for p, k in zip(plain, kept))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(kept[0].sum(), leaves[0])


@pytest.mark.parametrize("size", [6, 70])
def test_every_choice_of_wanted_gradients(cuda_device, size):
    x, dy, w, b = make((2, size, 10, 24), 3, F32, F32)
    everything = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(group_norm_act(everything[0], 3, everything[1], everything[2], eps=EPS), everything, dy)
    for mask in range(1, 7):
        leaves = [t.detach().requires_grad_(bool(mask >> k & 1)) for k, t in enumerate((x, w, b))]
        wanted = [k for k in range(3) if mask >> k & 1]
        got = torch.autograd.grad(group_norm_act(leaves[0], 3, leaves[1], leaves[2], eps=EPS), [leaves[k] for k in wanted], dy)
        assert all(torch.equal(g, want[k]) for g, k in zip(got, wanted))


def test_most_images(cuda_device):
    x, dy, w, b = make((65535, 2, 3), 3, F32, F32)
    check(x, dy, w, b, 3, "silu")


def test_refusals_on_the_device(cuda_device):
    x = torch.zeros(2, 3, 3, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for bad in (lambda: group_norm_act(x, 3, w), lambda: group_norm_act(x, 0, w), lambda: group_norm_act(x, 2, w[:4]),
                lambda: group_norm_act(x, 2, w.double()), lambda: group_norm_act(x.double(), 2, w),
                lambda: group_norm_act(x, 2, w.cpu()), lambda: group_norm_act(x, 2, w, w.half()),
                lambda: group_norm_act(x, 2, w, act="relu"), lambda: group_norm_act(x, 2, w, eps=-1.0), lambda: group_norm_act(x, 2, w, eps=1e300),
                lambda: group_norm_act(x, 2, w, eps=float("nan")), lambda: group_norm_act(x[0, 0, 0], 2, w)):
        with pytest.raises(ValueError, match="group_norm_act"):
            bad()
    with pytest.raises(RuntimeError, match="16385 channels"):
        group_norm_act(torch.zeros(1, 2, 16385, device="cuda"), 1)
