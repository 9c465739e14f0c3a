"""orthogonalize and muon_step where the products take 256-wide tiles: X X^T and A V from more than fifty tiles on the upper
triangle on, one matrix with a short side above 2304 or several smaller ones.  And what 16-bit operands cost."""
import pytest
import torch

from d3gs_research_b200 import orthogonalize
from test_gpu_muon import BF16, F32, NS, chain, check, check_step, make, tensors

pytestmark = pytest.mark.gpu


# odd and even numbers of 128-row blocks, short sides that end inside a block of 64, the long side on either axis
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n", [(2400, 2500), (2600, 2330), (2497, 2497), (3600, 2690)])
def test_one_large_matrix(cuda_device, m, n, dtype):
    check(make(m, n, seed=m).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_stacks_of_large_matrices(cuda_device, dtype):
    u = torch.stack([make(1100, 1300, seed=k) for k in range(5)]).to(dtype)
    got = check(u)
    assert torch.equal(orthogonalize(u), got)


def test_a_list_of_large_matrices(cuda_device):
    check_step(*tensors([(1100, 1300), (2048, 1500), (1300, 1090), (1700, 2000), (400, 1600), (60, 70)]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n", [(40, 60), (300, 200), (64, 2000), (500, 420), (450, 9000), (2400, 2500)])
def test_coefficients_without_a_fifth_power(cuda_device, m, n, dtype):
    """The first product gives B there; alone, and between steps that have all three."""
    u = make(m, n, seed=n).to(dtype)
    check(u, ns_coefficients=(1.5, -0.5, 0.0), ns_steps=6)
    check(u, ns_coefficients=[NS, (1.5, -0.5, 0.0), NS, (2.0, 0.0, 0.0), (1.2, -0.2, 0.0)], ns_steps=5)


def to_bits(v, bits):
    m, e = torch.frexp(v)
    return torch.ldexp(torch.round(m * 2.0 ** bits), e - bits)


def sixteen_bit_chain(u, planes):
    """The chain with the operands that products of 16-bit matrices have: A, V = A + b/c I on the diagonal, and B in 11
    bits, X as it is in the first step, then 11 bits of it in X X^T and ``planes[step]`` values of 11 in B X.  The upper
    triangle of A V stands for the lower one too."""
    x = u.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / torch.linalg.vector_norm(x)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    a, b, c = NS
    for step, p in enumerate(planes):
        first = x if step == 0 else to_bits(x, 11)
        gram = first @ first.T
        big = to_bits(gram, 11)
        v = big.clone()
        v.diagonal().copy_(to_bits(gram.diagonal() + b / c, 11))
        half = torch.triu(big @ v)
        poly = to_bits(a * eye + c * (half + torch.triu(half, 1).T), 11)
        x = poly @ (x if step == 0 else to_bits(x, 11 * p))
    return x.T if tall else x


@pytest.mark.parametrize("m,n", [(640, 640), (1100, 1030), (2400, 2500)])
def test_what_16_bit_operands_cost(cuda_device, m, n):
    """The output's own rounding is known (that of the exact result) and independent of what came before it, so the error
    before it is the square root of a difference of squares.  It may be a seventh above that of the same roundings done anew
    (another draw of them in hundreds of singular directions; tiles on the diagonal, which have both triangles; the tensor
    cores' sums, 2e-5); X in one value everywhere costs a third more at least, and would be noticed."""
    u = make(m, n, seed=m * 7 + n).to(BF16)
    ref = chain(u)
    size = torch.linalg.vector_norm(ref)
    off = lambda y: (torch.linalg.vector_norm(y.double() - ref) / size).item()   # noqa: E731
    cost, coarse = (off(sixteen_bit_chain(u, p)) for p in ((1, 2, 2, 2, 1), (1, 1, 1, 1, 1)))
    assert coarse > 1.3 * cost
    assert off(orthogonalize(u)) ** 2 - off(ref.to(BF16)) ** 2 <= (1.15 * cost) ** 2


@pytest.mark.parametrize("m,n", [(512, 2048), (1024, 1024), (2048, 4096)])
@pytest.mark.parametrize("coefs", [(1.0, -1.0, 0.0), (2.0, -3.0, 1.0)])
def test_the_low_half_of_x_is_in_every_entry(cuda_device, m, n, coefs):
    """16 bits: a matrix with one strong direction of equal entries, which the middle step takes out.  What is left was in
    the last bits of X: with the high half alone it is 6e-3 off or more, with both its own rounding (up to 1.7e-3) and a
    tenth.  Errors along the strong direction on either side, where A's rounding shows, are set aside.  Every 64 rows and
    columns are held to it."""
    g = torch.Generator(device="cuda").manual_seed(1)
    u = (torch.ones(m, n, device="cuda") + 2.0 ** -5 * torch.randn(m, n, generator=g, device="cuda")).to(BF16)
    steps = [(1.0, 0.0, 0.0), coefs, (1.0, 0.0, 0.0)]
    ref = chain(u, steps)
    err = orthogonalize(u, ns_coefficients=steps, ns_steps=3).double() - ref
    err = err - err.mean(0, keepdim=True) - err.mean(1, keepdim=True) + err.mean()
    rounding = torch.linalg.vector_norm(ref.to(BF16).double() - ref) / torch.linalg.vector_norm(ref)
    for axes, cut in (((0, 2), (m, n // 64, 64)), ((1, 2), (m // 64, 64, n))):
        share = (err.reshape(cut).square().sum(axes) / ref.reshape(cut).square().sum(axes)).sqrt()
        assert share.max() <= 1.1 * rounding
