"""Newton-Schulz orthogonalisation of matrices that its number format holds worst: equal singular values, rows of very different size, one value that
outweighs all others.  There an fp32 iteration can be nearly exact by chance, and the bounds come from the format alone.

A value v (of X, A or B) is held as f16 halves of 4096 v: off by at most 2^-22 |v| + 2^-37 (the lower half rounds by 2^-11 of the upper one's rounding,
or by half the smallest f16).  A product over K drops the product of the lower halves, 2^-22 of a sum of independent signs, and rounds its fp32
sum 3 K / 32 times by 2^-24: r(K) = 2^-22 + 3 K / 32 2^-24, to which the storage of the result adds 2^-22 (h below).  With s the singular values of X in one step and s1
the largest, in the Frobenius norm, to first order:
    A off by h(t) |A|       moves the next X by  (|b| + 2 |c| s1^2) s1 times that
    A A off by r(s) |A| s1^2     moves it by     |c| s1 times that,   the storage of B, 2^-22 |B|, by s1 times that
    B X off by r(s) |B| s1, and the storage of the next X by 2^-22 of its norm (and 2 more fp32 roundings: 2^-23)
    the 2^-37 of each element add 2^-37 (sqrt(s t) + s (|b| + 2 |c| s1^2 + 1) s1)
and what an earlier step left is multiplied by at most the largest divided difference of the polynomial over the singular values, mirrored at 0."""
import pytest
import torch

from acmil_amd import ops

pytestmark = pytest.mark.gpu
CO = (3.4445, -4.7750, 2.0315)


def iterate(g, steps=5, eps=1e-7):
    """the definition in 64 bits, and the bound above"""
    a, b, c = CO
    x = g.double().cpu()
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / (x.norm() + eps)
    s, t = x.shape
    r = lambda k: 2.0 ** -22 + 3 * k / 32 * 2.0 ** -24
    off = 2.0 ** -22 * float(x.norm()) + 2.0 ** -37 * (s * t) ** 0.5
    for k in range(steps):
        sv = torch.linalg.svdvals(x)
        s1, A, B = float(sv[0]), float((sv ** 2).norm()), float((b * sv ** 2 + c * sv ** 4).norm())
        both = torch.cat([sv, -sv])
        p = a * both + b * both ** 3 + c * both ** 5
        gap = both[:, None] - both[None, :]
        near = gap.abs() < 1e-6
        slope = a + 3 * b * both ** 2 + 5 * c * both ** 4
        grow = float(torch.where(near, slope.abs()[:, None].expand_as(gap), ((p[:, None] - p[None, :]) / torch.where(near, torch.ones_like(gap), gap)).abs()).max())
        q = x @ x.t()
        x = a * x + (b * q + c * (q @ q)) @ x
        off = grow * off + (r(t) + 2.0 ** -22) * A * (abs(b) + 2 * abs(c) * s1 ** 2) * s1 + r(s) * A * s1 ** 3 * abs(c) + (2.0 ** -22 + r(s)) * B * s1 \
            + (2.0 ** -22 + 2.0 ** -23) * float(x.norm()) + 2.0 ** -37 * ((s * t) ** 0.5 + s * (abs(b) + 2 * abs(c) * s1 ** 2 + 1) * s1)
    return (x.t() if tall else x), off


def check(g):
    want, bound = iterate(g)
    off = float((ops.orthogonalize(g).double().cpu() - want).norm())
    assert off <= bound, (off, bound)
    assert bound <= 2e-2 * float(want.norm())                          # a bound that means something


def normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# one workgroup (X within one CU's LDS), and tiles
SIZES = [(1, 40), (30, 100), (64, 64), (96, 200), (128, 161), (200, 96), (256, 256), (512, 768)]


@pytest.mark.parametrize("m, n", SIZES)
def test_equal_singular_values(m, n):
    check(torch.eye(m, n).cuda())
    q = torch.linalg.qr(normal(max(m, n), min(m, n), seed=m).double())[0].float()
    check((q if m >= n else q.t()).contiguous().cuda())


@pytest.mark.parametrize("m, n", SIZES)
def test_rows_and_columns_of_different_size(m, n):
    g = normal(m, n, seed=n)
    check((g * torch.logspace(0, -6, m)[:, None]).cuda())
    check((g * torch.logspace(0, -6, n)).cuda())


@pytest.mark.parametrize("m, n", [(30, 100), (120, 150), (100, 31), (200, 300), (300, 150)])
@pytest.mark.parametrize("outlier", [1e3, 1e5, 1e7, 1e9])
def test_one_value_outweighs_the_others(m, n, outlier):
    """The value stands alone in its row and column, so the rest iterates by itself: its values are so small that a step multiplies them by at most
    a = 3.4445, rounds them by 2^-22 + 2^-23 and moves each by 2^-37 when it is stored: what the format holds of small values, and no more."""
    g = torch.zeros(m, n)
    g[1:, 1:] = normal(m - 1, n - 1, seed=3)
    g[0, 0] = outlier * float(g.norm())
    want, _ = iterate(g)
    x = g.double() / (g.double().norm() + 1e-7)
    size, each = float(x[1:, 1:].norm()), 2.0 ** -37 * ((m - 1) * (n - 1)) ** 0.5
    off = 2.0 ** -22 * size + each
    for _ in range(5):
        size *= CO[0]
        off = CO[0] * off + (2.0 ** -22 + 2.0 ** -23) * size + each
    # what is left out above: A and B of the block, at most size^2 and 7 size^2 wide, and their 2^-37 an element, times the block
    off += 485 * (7 * 2.0 ** -20 * size ** 3 + 14 * 2.0 ** -37 * min(m, n) * size)
    got = ops.orthogonalize(g.cuda()).double().cpu()
    rest = (got - want)[1:, 1:]
    assert float(rest.norm()) <= off, (float(rest.norm()), off)
    assert abs(float(got[0, 0] - want[0, 0])) <= 1e-4 and not got[0, 1:].any() and not got[1:, 0].any()
