"""Newton-Schulz where values of very different size meet: rows, columns and
diagonals graded over many powers of ten, more steps than the default, and
matrices whose norm is small beside eps.  Compared with the 64-bit iteration
under the bound of test_gpu_newton_schulz, four times the distance of 32-bit
floats on the same input and 2^-20 of the result's norm, which is derived
there for operands that are rounded relative to their own size.

A diagonal matrix is a scalar iteration for each of its elements.  Its products
are of one term, in which 32-bit floats round once: they are no measure there,
and the error is bounded step by step instead.
"""

import pytest
import torch

from test_gpu_newton_schulz import MUON, check, matrix

pytestmark = pytest.mark.gpu


def graded(kind, m, n, power, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=gen)
    rows = torch.logspace(0, -power, m)[:, None]
    cols = torch.logspace(0, -power, n)[None]
    if kind == "rows":
        x = x * rows
    elif kind == "cols":
        x = x * cols
    elif kind == "both":
        x = x * rows * cols
    else:  # two blocks that have nothing to do with one another
        x[: m // 2, n // 2:] = 0.0
        x[m // 2:, : n // 2] = 0.0
        x[m // 2:] *= 10.0**-power
    return x.cuda()


# In one workgroup, as split tiles, tall, and 128 tiles of 256 x 128 or more.
SHAPES = [(100, 128), (128, 60), (16, 500), (200, 300), (300, 180)]


@pytest.mark.parametrize("steps", [5, 9, 12, 16])
@pytest.mark.parametrize("kind", ["rows", "cols", "both", "blocks"])
def test_graded(sporder, kind, steps):
    for shape in SHAPES:
        for power in (6, 8):
            g = graded(kind, *shape, power, seed=steps)
            check(sporder.newton_schulz(g, steps=steps), g, steps)


def diagonal_bound(start, steps, n, eps=1e-7):
    """The iteration on a diagonal in 64 bits, and a bound on each element's
    error, to first order.

    u = 2^-24 is a 32-bit rounding.  An operand of two halves is off by 2u of
    itself and, as a half's last step is 2^-24 and its row's unit 2^-14 of the
    row's bound r at most, by 2^-39 r; r is at most the element times sqrt(n)
    and the maximum g = a of |a + b t + c t^2| to the power of the steps, and at
    most S < 1.25.  A's unit is S's power of two, 2, times X's, B's at most 4
    times (h = max |s (b + c s^2)| < 2.4).  A product is off by 2u for each
    operand, 4u for the low halves' product that is left out and 2u for its
    additions: 10u.  Coefficients are rounded once."""
    a, b, c = MUON
    u = 2.0**-24
    s0 = start.double()
    s = s0 / (s0.norm() + eps)
    off = u * s
    for k in range(steps):
        r = torch.clamp(s0 / (s0.norm() + eps) * n**0.5 * 1.01 * a**k, max=1.25)
        floor = 2.0**-39 * r
        gram = s * s
        d_gram = 10 * u * gram + 2 * floor * s
        held = d_gram + 2 * u * gram + 2 * floor  # as an operand
        poly = b * gram + c * gram * gram
        d_poly = (abs(b) * (held + 3 * u * gram)
                  + c * (2 * held * gram + 10 * u * gram * gram + 3 * u * gram * gram))
        update = poly * s
        d_update = ((d_poly + 2 * u * poly.abs() + 4 * floor) * s + poly.abs() * (2 * u * s + floor)
                    + 6 * u * update.abs())
        new = a * s + update
        slope = (a + 3 * b * gram + 5 * c * gram * gram).abs()
        off = slope * off + d_update + 3 * u * a * s + u * (a * s + update.abs())
        s = new
    return s, 1.05 * off


@pytest.mark.parametrize("steps", [5, 9, 12, 16])
def test_diagonals(sporder, steps):
    for shape in SHAPES:
        for power in (0, 3, 6, 8):
            k = min(shape)
            start = torch.logspace(0, -power, k)
            g = torch.zeros(shape)
            g[torch.arange(k), torch.arange(k)] = start
            got = sporder.newton_schulz(g.cuda(), steps=steps).cpu()
            want, bound = diagonal_bound(start, steps, max(shape))
            assert ((torch.diagonal(got).double() - want).abs() <= bound).all()
            assert bound.max() < 0.05  # or it says nothing
            got[torch.arange(k), torch.arange(k)] = 0.0
            assert not got.any()


@pytest.mark.parametrize("kind", ["rows", "cols"])
def test_graded_in_large_tiles(sporder, kind):
    from test_gpu_newton_schulz_large import iterate
    g = graded(kind, 2049, 2304, 8, seed=1)
    got = sporder.newton_schulz(g, steps=12)
    exact = iterate(g, torch.float64, 12)
    plain = (iterate(g, torch.float32, 12).double() - exact).norm()
    assert (got.double() - exact).norm() <= 4 * plain + 2.0**-20 * exact.norm()


@pytest.mark.parametrize("size", [1e-5, 1e-9, 1e-14, 1e-17, 1e-25, 1e-35])
def test_norm_below_eps(sporder, size):
    for shape in SHAPES + [(300, 700)]:
        g = matrix(*shape, seed=11)
        g = g * (size / g.norm())
        check(sporder.newton_schulz(g), g)
        check(sporder.newton_schulz(g, steps=9), g, 9)


@pytest.mark.parametrize("coefficients,steps", [((1.5, -0.5, 0.0), 25), ((1.5, -0.5, 0.0), 60),
                                                ((2.0, 0.0, 0.0), 3), ((0.5, 0.0, 0.0), 20),
                                                ((0.0, 0.0, 0.0), 2), ((0.0, 1.0, 0.0), 2),
                                                ((5.0, 1.0, 1.0), 1)])
def test_graded_under_other_coefficients(sporder, coefficients, steps):
    for shape in SHAPES:
        g = graded("rows", *shape, 6, seed=steps)
        got = sporder.newton_schulz(g, steps=steps, coefficients=coefficients)
        check(got, g, steps, coefficients)
