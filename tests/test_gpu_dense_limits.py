"""The dense operators at the ends of what they accept."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8


@pytest.mark.parametrize("m,n", [(1, 1), (40, 72), (300, 136)])
def test_polynomials_near_the_largest_singular_value(et, dev, m, n):
    """1.07 a step and nothing else: a matrix of rank one, whose singular value is 1, ends at 1.07^6 = 1.50.  X and S are
    rounded to f16 before each of the 6 products and X behind the last (13 half steps of 2^-11), and to bf16 once."""
    g = torch.Generator(device=dev).manual_seed(m + n)
    u = torch.randn(2, m, 1, generator=g, device=dev) * torch.randn(2, 1, n, generator=g, device=dev)
    got = et.orthogonalize(u, steps=6, coefficients=(1.07, 0.0, 0.0), eps=0.0).double()
    want = u.double() / u.double().flatten(1).norm(dim=1)[:, None, None] * 1.07 ** 6
    off = ((got - want).flatten(1).norm(dim=1) / 1.07 ** 6).max().item()
    assert off <= 13 * 2.0 ** -11 + HALF, off
