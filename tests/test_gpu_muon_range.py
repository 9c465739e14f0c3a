"""orthogonalize and muon_step over long lists, and at the ends of the floats' range: norms and eps whose reciprocals a 32-bit float does not
hold.  On every way through the products: a CTA a matrix, tiles, pairs of CTAs, shared sums."""
import pytest
import torch

from d3gs_research_b200 import muon_step, orthogonalize
from test_gpu_muon import BF16, F32, check, check_step, make, tensors

pytestmark = pytest.mark.gpu

ROUTES = [(40, 60), (200, 300), (300, 70), (500, 420), (500, 8200)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n", ROUTES)
def test_zeros_stay_zeros_whatever_eps(cuda_device, m, n, dtype):
    u = torch.zeros(m, n, dtype=dtype, device="cuda")
    for eps in (2.0 ** -149, 2.0 ** -127, 1e-37, 1e-20, 1e38):
        got = orthogonalize(u, eps=eps)
        assert not got.any() and not torch.isnan(got).any()


@pytest.mark.parametrize("m,n", ROUTES)
def test_a_layer_without_gradient_only_decays(cuda_device, m, n):
    p = torch.randn(m, n, device="cuda")
    want = p.double() * (1 - 0.1 * 0.5)
    g, buf = torch.zeros_like(p), torch.zeros_like(p)
    muon_step([p], [g], [buf], lr=0.1, weight_decay=0.5, eps=2.0 ** -140)
    # decay rounded to 32 bits, and the product
    assert ((p.double() - want).abs() <= 2 * 2.0 ** -24 * want.abs()).all()
    assert not buf.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n", ROUTES)
def test_very_small_and_very_large_updates(cuda_device, m, n, dtype):
    """Powers of two, so that what scaling rounds is in the input: norms of about 2^-135 (entries below the normal range),
    2^-120 and beyond 2^128.  eps is a 32-bit float."""
    u = make(m, n, scale=1.0)
    u = u / u.abs().max()
    check((u * 2.0 ** -138).to(dtype), eps=2.0 ** -149)
    check((u * 2.0 ** -126).to(dtype), eps=2.0 ** -149)
    check((u * 2.0 ** -126).to(dtype), eps=2.0 ** -112)      # far below eps
    check((u * 1.99 * 2.0 ** 127 * 0.99).to(dtype))
    check((u * 2.0 ** 100).to(dtype), eps=2.0 ** 120)


def launches(call):
    from d3gs_research_b200 import _lib
    lib = _lib.load()
    before = lib.d3gs_kernel_launch_count()
    call()
    return lib.d3gs_kernel_launch_count() - before


def test_long_lists_take_their_workspace_and_their_way_a_batch(cuda_device):
    """Eighty tiny matrices with one large among them, and forty large ones with tiny ones between: every result is that of
    the formula, and what a batch of 32 has left of the tiny ones takes a launch a batch."""
    for shapes, most in (([(8 + k % 5, 16 + k % 40) for k in range(80)] + [(500, 420)], 18 + 2),
                         ([(400, 390 + k // 2) if k % 2 else (8, 16 + k) for k in range(80)], 2 * 18 + 1)):
        run = tensors(shapes)
        assert launches(lambda: check_step(*run)) == most
    u = torch.stack([make(24, 40, seed=k) for k in range(100)])
    assert launches(lambda: orthogonalize(u)) == 4
    check(u)
    for dtype in (F32, BF16):      # the workspace of one batch after another, no stale values in it
        v = torch.stack([make(390 + 2, 500, seed=k) for k in range(40)]).to(dtype)
        got = check(v)
        assert torch.equal(orthogonalize(v[35]), orthogonalize(v[35:36])[0])
        assert torch.equal(orthogonalize(v), got)


@pytest.mark.parametrize("m,n,dtype", [(40, 1000003, F32), (1000003, 40, BF16), (500, 80000, F32)])
def test_so_many_values_that_a_cta_takes_several_turns_of_the_norm(cuda_device, m, n, dtype):
    check(make(m, n).to(dtype))


def test_step_of_so_many_values(cuda_device):
    check_step(*tensors([(40, 900001), (30, 20)]))


@pytest.mark.parametrize("mu", [0.0, 0.3, 0.95, 0.999, 0.9999, 1 - 2.0 ** -20])
@pytest.mark.parametrize("m,n", [(40, 60), (300, 200), (500, 420)])
def test_the_gradients_weight_is_one_minus_the_momentum(cuda_device, m, n, mu):
    """1 - mu as the difference of 64-bit numbers: the difference of 32-bit ones is 1e-3 off for a momentum near one.  Two
    roundings of the new buffer: the weight's and the product's; with an old one, three, each of at most the terms' size."""
    g, old = make(m, n, seed=1), make(m, n, seed=2)
    for start in (torch.zeros_like(old), old):
        buf = start.clone()
        muon_step([torch.zeros(m, n, device="cuda")], [g], [buf], lr=0.1, momentum=mu)
        kept, fresh = mu * start.double(), (1 - mu) * g.double()
        assert ((buf.double() - kept - fresh).abs() <= 3 * 2.0 ** -24 * (kept.abs() + fresh.abs()) + 2.0 ** -149).all()


def test_the_updates_weights_are_those_of_the_buffer(cuda_device):
    """Nesterov: the update mu buffer + (1 - mu) g.  With an old buffer of zeros the update is (1 - mu^2) g, with a momentum of
    zero g; with a buffer far from the gradient the weights show in the direction."""
    for mu in (0.0, 0.95, 0.9999):
        run = tensors([(40, 60), (300, 200), (500, 420)])
        run[1][:] = [1e3 * g for g in run[1]]
        check_step(*run, mu=mu)
