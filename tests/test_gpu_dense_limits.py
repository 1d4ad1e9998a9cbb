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


@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,m,n", [(3, 8, 16), (3, 64, 1024), (3, 500, 40), (3, 130, 77), (40, 384, 520)])
def test_a_zero_matrix_gives_zero_without_eps(et, dev, E, m, n, dtype, eps):
    """By every way that a matrix can go; a bad matrix and others beside it (eps 1e-60 is 0 in binary32)."""
    g = torch.randn(E, m, n, generator=torch.Generator(device=dev).manual_seed(m), device=dev).to(dtype)
    want = et.orthogonalize(g, eps=eps)
    assert torch.isfinite(want.float()).all() and want.any()
    g[1] = 0
    got = et.orthogonalize(g, eps=eps)
    assert not got[1].any()
    assert torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])
    for bad in (float("nan"), float("inf")):
        g[2, m // 2, n // 3] = bad
        got = et.orthogonalize(g, eps=eps)
        assert not got[1].any() and bool(torch.isnan(got[2]).all()) and torch.equal(got[0], want[0])


@pytest.mark.parametrize("m,n", [(16, 64), (96, 264)])
@pytest.mark.parametrize("low", [False, True])
def test_an_expert_without_tokens_keeps_its_weights(et, dev, m, n, low):
    """A step without eps, the second expert's gradient and momentum zero: its weights decay and stay."""
    g = torch.randn(3, m, n, generator=torch.Generator(device=dev).manual_seed(n), device=dev)
    g[1] = 0
    w = torch.ones_like(g)
    params = [w.bfloat16() if low else w]
    masters = [w] if low else None
    momenta = [torch.zeros_like(g)]
    et.muon_step_(params, [g], momenta, lr=0.5, weight_decay=0.5, eps=0.0, masters=masters)
    assert bool((w[1] == 0.75).all()) and bool((params[0][1] == 0.75).all()) and not momenta[0][1].any()
    assert torch.isfinite(w).all() and bool((w[0] != 0.75).any())


def test_more_small_matrices_than_a_launch_takes(et, dev):
    """Two tensors of 2^22 + 5 matrices of one row, a block each: more than 2^23 blocks in all.  A row's singular
    value is 1 and follows the polynomial; X and S are rounded to f16 in 5 steps (a factor of up to 3.45 in the first, below
    1 in size behind it: 5 products of 3 roundings each, times 3.45), and to bf16 once in one of the calls."""
    E = (1 << 22) + 5
    g = torch.Generator(device=dev).manual_seed(8)
    us = [torch.randn(E, 1, n, generator=g, device=dev) + 3.0 for n in (1, 2)]
    ps, moms = [torch.zeros_like(u) for u in us], [torch.zeros_like(u) for u in us]
    et.muon_step_(ps, us, moms, lr=1.0, momentum=0.0, nesterov=False, update_rms=None)
    s = 1.0
    for _ in range(5):
        s = s * (3.4445 - 4.7750 * s ** 2 + 2.0315 * s ** 4)
    for u, p, m in zip(us, ps, moms):
        assert torch.equal(m, u)
        want = u.double() / u.double().flatten(1).norm(dim=1)[:, None, None] * s
        assert ((-p.double() - want).abs().amax() <= 15 * 3.45 * 2.0 ** -11).item()
