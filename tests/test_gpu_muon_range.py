"""orthogonalize and muon_step at the ends of the floats' range: norms and eps whose reciprocals a 32-bit float does not
hold.  On every way through the products: a CTA a matrix, tiles, pairs of CTAs, shared sums."""
import pytest
import torch

from d3gs_research_b200 import muon_step, orthogonalize
from test_gpu_muon import BF16, F32, check, make

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
