"""orthogonalize, muon_step and GaussianMuon against their formulas in 64 bits.

Tolerance.  A Newton-Schulz step multiplies a small singular value, and with it every earlier rounding in its
direction, by up to 3.4, so what a rounding costs depends on the matrix.  ``chain`` therefore runs the 64-bit
formula a second time with every operand of every product rounded to ``bits`` bits (with a random sign): the
distance between the two runs is what arithmetic of that width costs on this matrix.  32-bit matrices are held to
four times the cost of 20 bits (operands of 22 bits, and sums whose last bits are lost over long rows), 16-bit ones
to four times the cost of 11 bits, both in the 2-norm, plus half a step of the output's type.  Operands are fp16 values
of a scale of 2^15, whose smallest step is 2^-24: an entry of X is off by 2^-25 / 2^15 = 2^-40 at least, and a small
singular value, with the error in its direction, grows by the product of the steps' a.
"""
import copy
import math

import pytest
import torch

from d3gs_research_b200 import GaussianMuon, muon_step, orthogonalize

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)
F32, BF16 = torch.float32, torch.bfloat16


def chain(u, coefs=(NS,) * 5, eps=1e-7, bits=None):
    gen = torch.Generator(device="cuda").manual_seed(99)

    def rounded(v):
        if bits is None:
            return v
        return v * (1 + 2.0 ** -bits * (2 * torch.rand(v.shape, generator=gen, device="cuda", dtype=torch.float64) - 1))

    x = u.double()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    x = rounded(x / max(torch.linalg.vector_norm(x).item(), eps))
    for a, b, c in coefs:
        gram = rounded(x @ x.T)
        poly = rounded(b * gram + c * (gram @ gram))
        x = rounded(a * x + poly @ x)
    return x.T if tall else x


def bound(u, ref, dtype, coefs=(NS,) * 5, eps=1e-7):
    cost = torch.linalg.vector_norm(chain(u, coefs, eps, 20 if dtype == F32 else 11) - ref)
    return 4 * cost + torch.finfo(dtype).eps / 2 * torch.linalg.vector_norm(ref) \
        + 4 * math.sqrt(u.numel()) * 2.0 ** -40 * math.prod(max(1.0, abs(c[0])) for c in coefs)


def make(m, n, seed=0, scale=1e-3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = max(1, min(m, n) // 4)
    u = torch.randn(m, r, generator=g, device="cuda") @ torch.randn(r, n, generator=g, device="cuda")
    return scale * (u + 0.3 * math.sqrt(r) * torch.randn(m, n, generator=g, device="cuda"))


def check(u, what="", **kw):
    got = orthogonalize(u, **kw)
    assert got.shape == u.shape and got.dtype == u.dtype and got.is_contiguous()
    coefs = kw.get("ns_coefficients", NS)
    steps = kw.get("ns_steps", 5)
    coefs = coefs if isinstance(coefs[0], tuple) else (coefs,) * steps
    eps = kw.get("eps", 1e-7)
    for v, w in zip(u.reshape(-1, *u.shape[-2:]), got.reshape(-1, *u.shape[-2:])):
        ref = chain(v, coefs, eps)
        err = torch.linalg.vector_norm(w.double() - ref)
        assert err <= bound(v, ref, u.dtype, coefs, eps), \
            f"{what} {tuple(u.shape)}: {err.item()} of {torch.linalg.vector_norm(ref).item()}"
    return got


SIZES = [(1, 1), (1, 7), (5, 1), (2, 2), (3, 64), (64, 64), (65, 63), (127, 129), (128, 128), (129, 1000), (128, 8), (257, 255),
         (300, 70), (512, 192), (200, 1111), (1111, 130), (64, 4000), (1, 5000), (640, 640), (1025, 515),
         (385, 400), (500, 1300), (700, 2100), (20, 192), (128, 256), (256, 100), (77, 257), (129, 128), (100, 192), (192, 128), (100, 193)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n", SIZES)
def test_sizes(cuda_device, m, n, dtype):
    check(make(m, n, seed=m * 7 + n).to(dtype))


@pytest.mark.parametrize("m,n,dtype", [(2048, 1500, F32), (1500, 2048, BF16), (96, 16384, F32), (4096, 256, BF16),
                                       (500, 8200, F32), (8200, 500, BF16), (1000, 4200, F32), (450, 20000, BF16)])
def test_large_sizes(cuda_device, m, n, dtype):
    check(make(m, n).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_stacks(cuda_device, dtype):
    """More matrices than one launch takes, two leading axes, and the same result as one by one."""
    u = torch.stack([make(24, 40, seed=k) for k in range(150)]).to(dtype)
    got = check(u)
    assert torch.equal(orthogonalize(u[70]), got[70])
    assert torch.equal(orthogonalize(u.view(10, 15, 24, 40)).view_as(got), got)
    check(torch.stack([make(300, 140, seed=k) for k in range(5)]).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(cuda_device, dtype):
    u = make(70, 90).to(dtype)
    base = check(u)
    wide = torch.zeros(75, 101, dtype=dtype, device="cuda")
    wide[3:73, 5:95] = u
    assert torch.equal(orthogonalize(wide[3:73, 5:95]), base)
    assert torch.equal(orthogonalize(u.T.contiguous().T), base)
    assert torch.equal(orthogonalize(torch.stack([u, u])[:, :, :][::1].transpose(0, 1).contiguous().transpose(0, 1))[1], base)
    check(wide[::3, ::2][:20])
    check(u[:1].expand(70, 90))
    check(u[:, :1])


def test_steps_and_coefficients(cuda_device):
    u = make(90, 120)
    for steps in (1, 2, 7):
        check(u, ns_steps=steps)
    check(u, ns_coefficients=(2.0, -1.5, 0.5), ns_steps=8)
    check(u, ns_coefficients=[(4.0, -6.0, 2.8), (3.0, -3.4, 1.2), (2.0, -1.5, 0.5)], ns_steps=3)
    check(u, ns_coefficients=(1.5, -0.5, 0.0), ns_steps=12)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_magnitudes(cuda_device, dtype):
    """Squares that a 32-bit sum would overflow or lose; a norm below eps; rows of very different size."""
    u = make(60, 100, scale=1.0)
    check((u * 1e30).to(dtype))
    check((u * 1e-25).to(dtype), eps=1e-30)
    check((u * torch.logspace(0, -6, 60, device="cuda")[:, None]).to(dtype))
    small = (u * 1e-10).to(dtype)              # X = U / eps stays small: nothing is amplified to one
    check(small, eps=1e-2)
    assert not orthogonalize(torch.zeros(33, 20, dtype=dtype, device="cuda")).any()


def test_one_strong_direction_and_orthogonal_input(cuda_device):
    g = torch.Generator(device="cuda").manual_seed(1)
    u = torch.randn(80, 1, generator=g, device="cuda") @ torch.randn(1, 140, generator=g, device="cuda")
    check(u)
    q = torch.linalg.qr(torch.randn(150, 90, generator=g, device="cuda"))[0]
    check(q)
    check(torch.eye(200, device="cuda"))
    spike = torch.full((64, 200), 1e-6, device="cuda")
    spike[3, 7] = 1.0
    check(spike)


def test_non_finite_values_spoil_their_matrix_only(cuda_device):
    for bad in (float("nan"), float("inf")):
        u = torch.stack([make(40, 150, seed=k) for k in range(3)])
        u[1, 7, 9] = bad
        got = orthogonalize(u)
        assert torch.isnan(got[1]).all()
        for k in (0, 2):
            assert torch.equal(got[k], orthogonalize(u[k]))


def test_empty(cuda_device):
    for shape in ((0, 5), (5, 0), (0, 4, 4)):
        assert orthogonalize(torch.empty(shape, device="cuda")).shape == shape
    muon_step([], [], [], lr=0.1)
    p = torch.empty(4, 0, device="cuda")
    muon_step([p], [p.clone()], [p.clone()], lr=0.1)


# ---- the step -------------------------------------------------------------------------------------------------
def reference_step(p, g, buf, lr, wd, mu, nesterov, adjust):
    rows = p.shape[0]
    flat = lambda t: t.double().reshape(rows, -1)   # noqa: E731
    buf64 = mu * flat(buf) + (1 - mu) * flat(g)
    u = mu * buf64 + (1 - mu) * flat(g) if nesterov else buf64
    cols = u.shape[1]
    ratio = 0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw" else math.sqrt(max(1, rows / cols))
    o = chain(u)
    return ((1 - lr * wd) * flat(p) - lr * ratio * o).reshape(p.shape), buf64.reshape(p.shape), o, u, lr * ratio


def check_step(params, grads, buffers, lr=0.02, wd=0.1, mu=0.95, nesterov=True, adjust=None):
    want = [reference_step(p, g, b, lr, wd, mu, nesterov, adjust) for p, g, b in zip(params, grads, buffers)]
    kept = [g.clone() for g in grads]
    muon_step(params, grads, buffers, lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov, adjust_lr_fn=adjust)
    for p, g, b, k, (rp, rb, o, u, rate) in zip(params, grads, buffers, kept, want):
        assert torch.equal(g, k)
        # three roundings of the buffer; two of the parameter, and the update's own error times its rate
        assert ((b.double() - rb).abs() <= 4 * 2.0 ** -24 * (rb.abs() + g.double().abs())).all()
        err = torch.linalg.vector_norm(p.double() - rp)
        assert err <= rate * bound(u, o, F32) + 3 * 2.0 ** -24 * torch.linalg.vector_norm(rp) \
            + 2.0 ** -23 * rate * torch.linalg.vector_norm(o)


SHAPES = [(64, 32), (3, 64), (64, 64), (128, 576), (70, 315), (33, 1), (1, 9), (600, 130), (64, 32, 3, 3), (20, 6, 5)]


def tensors(shapes, seed=0):
    out = ([], [], [])
    for k, s in enumerate(shapes):
        flat = (s[0], math.prod(s[1:]))
        out[0].append((make(*flat, seed=seed + 3 * k, scale=0.1)).reshape(s))
        out[1].append((make(*flat, seed=seed + 3 * k + 1, scale=1e-4)).reshape(s))
        out[2].append((make(*flat, seed=seed + 3 * k + 2, scale=1e-4)).reshape(s))
    return out


@pytest.mark.parametrize("nesterov,wd,adjust", [(True, 0.1, None), (False, 0.0, "match_rms_adamw"), (True, 0.0, "original")])
def test_step(cuda_device, nesterov, wd, adjust):
    check_step(*tensors(SHAPES), wd=wd, nesterov=nesterov, adjust=adjust)


def test_step_of_more_matrices_than_a_launch_takes(cuda_device):
    check_step(*tensors([(8 + k % 5, 16 + k) for k in range(70)]))


def test_step_of_long_and_short_matrices(cuda_device):
    """The long ones' sums over the long axis are shared among CTAs; the short ones in the same launch leave most of
    those without a column block.  The same bits every time."""
    shapes = [(512, 8192), (400, 30), (8200, 390), (3, 500)]
    runs = [tensors(shapes) for _ in range(3)]
    check_step(*runs[0])
    for run in runs[1:]:
        muon_step(*run, lr=0.02)
        assert all(torch.equal(a, b) for a, b in zip(run[0], runs[0][0]))


def test_step_layouts(cuda_device):
    """Channels-last filters, gradients of other strides than their parameter's."""
    params, grads, buffers = tensors([(32, 8, 3, 3), (40, 30), (40, 30), (16, 8, 1, 1)])
    cl = torch.channels_last
    params[0], buffers[0] = params[0].to(memory_format=cl), buffers[0].to(memory_format=cl)
    grads[1] = grads[1].T.contiguous().T
    grads[2] = torch.cat([grads[2], grads[2]], 1)[:, :30]
    grads[3] = grads[3].to(memory_format=cl)
    # columns in another order: the result has them in that order too
    want = [t.clone(memory_format=torch.contiguous_format) for t in (params[0], grads[0], buffers[0])]
    check_step(params, grads, buffers)
    check_step(*[[t] for t in want])
    assert torch.linalg.vector_norm(params[0] - want[0]) <= 1e-5 * torch.linalg.vector_norm(want[0])


def test_optimizer(cuda_device):
    """Three steps of two groups against the formula step by step; a parameter without a gradient; state_dict."""
    params, _, _ = tensors([(64, 48), (10, 64), (5, 5)])
    leaves = [torch.nn.Parameter(p) for p in params]
    opt = GaussianMuon([{"params": leaves[:1]}, {"params": leaves[1:], "lr": 0.05, "nesterov": False}], lr=0.02, weight_decay=0.01)
    bufs = [torch.zeros_like(p) for p in params]
    idle = leaves[2].detach().clone()
    for step in range(3):
        want = []
        for k, p in enumerate(leaves[:2]):
            p.grad = make(*p.shape, seed=50 + 2 * step + k)
            want.append(reference_step(p.detach(), p.grad, bufs[k], 0.05 if k else 0.02, 0.01, 0.95, k == 0, None))
        version = leaves[0]._version
        assert opt.step(lambda: torch.tensor(2.0)).item() == 2.0
        assert leaves[0]._version > version
        for k, (rp, rb, o, u, rate) in enumerate(want):
            bufs[k] = opt.state[leaves[k]]["momentum_buffer"].clone()
            assert torch.linalg.vector_norm(leaves[k].double() - rp) <= rate * bound(u, o, F32) + 1e-6 * torch.linalg.vector_norm(rp)
    assert torch.equal(leaves[2], idle) and len(opt.state) == 2
    twin = [torch.nn.Parameter(p.detach().clone()) for p in leaves]
    other = GaussianMuon([{"params": twin[:1]}, {"params": twin[1:]}])
    other.load_state_dict(copy.deepcopy(opt.state_dict()))     # loading alone would share the buffers
    for a, b in zip(leaves[:2], twin):
        a.grad = make(*a.shape, seed=77)
        b.grad = a.grad.clone()
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(leaves, twin))


def test_long_matrices_on_two_streams_and_in_graphs(cuda_device):
    """Sums that CTAs leave to one another: two streams and two graphs at once, each several times."""
    updates = [make(512, 8192, seed=1), make(8200, 400, seed=2)]
    want = [orthogonalize(u) for u in updates]
    graphs = []
    for u in updates:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = orthogonalize(u)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in updates]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, u, (graph, out) in zip(streams, updates, graphs):
            out.zero_()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(orthogonalize(u))
                graph.replay()
        torch.cuda.synchronize()
        for g, (graph, out), w in zip(got, graphs, want):
            assert torch.equal(g, w) and torch.equal(out, w)


def test_streams_and_graphs(cuda_device):
    """The same bits on another stream and from a captured graph, replayed twice on changing gradients; two graphs at
    once on two streams."""
    runs = []
    for seed in (0, 300):
        eager, graphed = tensors(SHAPES[:6], seed), tensors(SHAPES[:6], seed)
        muon_step(*tensors(SHAPES[:6], seed), lr=0.02)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            muon_step(*graphed, lr=0.02)
            out = orthogonalize(graphed[1][3])
        runs.append((eager, graphed, graph, out, seed))
    for k in range(2):
        for eager, graphed, graph, out, seed in runs:
            new = tensors(SHAPES[:6], seed + 40 * k)[1]
            for a, b, n in zip(eager[1], graphed[1], new):
                a.copy_(n)
                b.copy_(n)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in runs]
        for s, run in zip(streams, runs):
            with torch.cuda.stream(s):
                run[2].replay()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for run in runs:
                muon_step(*run[0], lr=0.02)
        torch.cuda.synchronize()
        for eager, graphed, graph, out, seed in runs:
            for a, b in zip(eager, graphed):
                assert all(torch.equal(p, q) for p, q in zip(a, b))
            assert torch.equal(out, orthogonalize(graphed[1][3]))


def test_refusals(cuda_device):
    u = torch.zeros(4, 6, device="cuda")
    for bad in (lambda: orthogonalize(u.half()), lambda: orthogonalize(u[0]), lambda: orthogonalize(u, ns_steps=0),
                lambda: orthogonalize(u, ns_steps=33), lambda: orthogonalize(u, eps=0.0),
                lambda: orthogonalize(u, ns_coefficients=(1.0, 2.0)), lambda: orthogonalize(u, ns_coefficients=[NS] * 4),
                lambda: orthogonalize(u, ns_coefficients=(1.0, float("nan"), 0.0))):
        with pytest.raises(ValueError, match="orthogonalize"):
            bad()
    a, b, c = (torch.zeros(4, 6, device="cuda") for _ in range(3))
    for args, kw in ((([a], [b], []), {}), (([a], [b], [c]), {"momentum": 1.0}), (([a], [b], [c]), {"lr": -1.0}), (([a], [b], [c]), {"lr": 1e300}),
                     (([a], [b], [c]), {"adjust_lr_fn": "x"}), (([a, a], [b, b], [c, c.clone()]), {}),
                     (([a, b], [b, b], [c, c]), {}), (([a], [b], [a]), {}), (([a[0]], [b[0]], [c[0]]), {}),
                     (([a.T], [b.T], [c.T]), {}), (([a], [b.half()], [c]), {}), (([a], [b.cpu()], [c]), {}),
                     (([a[:, :3]], [b[:, :3]], [c[:, :3]]), {}), (([a], [b.T], [c]), {})):
        with pytest.raises(ValueError, match="muon_step"):
            muon_step(*args, **{"lr": 0.1, **kw})
    # a gradient that shares memory with a parameter or a buffer, its own or another's, by one value or as a whole
    flat = torch.zeros(100, device="cuda")
    p, q, s, r = (flat[24 * k:24 * k + 24].view(4, 6) for k in range(4))
    for args in (([p], [p], [q]), ([p], [q], [q]), ([p, s], [a, s], [b, c]), ([p, a], [b, flat[23:47].view(4, 6)], [r, c]),
                 ([q], [flat[1:25].view(4, 6)], [s]), ([p], [flat[18:].as_strided((4, 6), (20, 1))], [s])):
        with pytest.raises(ValueError, match="gradient overlaps"):
            muon_step(*args, lr=0.1)
    muon_step([p, r], [q, q], [s, a], lr=0.1)          # neighbours, and one gradient for two parameters
    with pytest.raises(ValueError, match="GaussianMuon"):
        GaussianMuon([torch.nn.Parameter(torch.zeros(3, device="cuda"))])
    with pytest.raises(RuntimeError, match="singular values grow"):
        orthogonalize(u, ns_coefficients=(9.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="short side"):
        orthogonalize(torch.empty(16385, 1, device="cuda").expand(16385, 16385))


@pytest.mark.parametrize("m,n", [(50, 200), (200, 300), (500, 520), (500, 8200)])
def test_a_wait_that_gives_up_spoils_the_result_and_no_more(cuda_device, m, n):
    """One CTA of every product never asks for its first tile (nothing is in flight when its waits run out): the call
    returns, its result is NaN, and the next call is right."""
    from d3gs_research_b200 import _lib
    lib = _lib.load()
    u = make(m, n)
    want = orthogonalize(u)
    lib.d3gs_test_hooks(300, 0)
    try:
        got = orthogonalize(u)
        torch.cuda.synchronize()
    finally:
        lib.d3gs_test_hooks(0, -1)
    assert torch.isnan(got).all()
    assert torch.equal(orthogonalize(u), want)
