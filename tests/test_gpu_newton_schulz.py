"""Newton-Schulz orthogonalisation against the iteration in 64 bits.

Bounds.  The iteration amplifies an error like it amplifies the matrix, so
what counts is how large the elementary errors are beside those of the same
iteration in 32-bit floats, whose distance from the 64-bit result is measured
here on the same input: an operand of 22 bits and a sign is off by at most
2^-23 of its value (four times a 32-bit float's 2^-24 with the left-out product
of the low halves, 2^-22), and the sums are 32-bit ones on both sides.  So at
most four times that distance, 2^-20 of the result's norm on top for inputs
on which 32-bit floats happen to be exact, and one rounding to the type.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

R = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
MUON = (3.4445, -4.7750, 2.0315)


def iterate(g, steps, coefficients, eps, dtype):
    """The formula in `dtype` on the CPU."""
    x = g.cpu().to(dtype)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t().contiguous()
    a, b, c = coefficients
    x = x / ((x.double() ** 2).sum().sqrt() + eps).to(dtype)
    for _ in range(steps):
        gram = x @ x.t().contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t().contiguous() if tall else x


def check(got, g, steps=5, coefficients=MUON, eps=1e-7):
    assert got.shape == g.shape and got.dtype == g.dtype
    exact = iterate(g, steps, coefficients, eps, torch.float64)
    off = (got.cpu().double() - exact).norm()
    plain = (iterate(g, steps, coefficients, eps, torch.float32).double() - exact).norm()
    bound = 4 * plain + (2.0**-20 + R[g.dtype]) * exact.norm()
    assert off <= bound, (float(off), float(plain), float(exact.norm()))


def matrix(*shape, dtype=torch.float32, seed=0, rank=None):
    gen = torch.Generator().manual_seed(seed)
    if rank:
        x = torch.randn(*shape[:-1], rank, generator=gen) @ torch.randn(rank, shape[-1],
                                                                       generator=gen)
        x = x + 0.1 * torch.randn(*shape, generator=gen)
    else:
        x = torch.randn(*shape, generator=gen)
    return (1e-3 * x).to(dtype).cuda()


SHAPES = [(1, 1), (1, 7), (7, 1), (1, 3000), (3, 5), (5, 3), (31, 33), (33, 65), (64, 64),
          (100, 128), (128, 100), (128, 47), (127, 128), (128, 128), (129, 257), (16, 2000),
          (2000, 16), (200, 1000), (1000, 200), (512, 512), (700, 1300), (1300, 700), (1100, 1024)]


@pytest.mark.parametrize("shape", SHAPES)
def test_shapes_and_types(sporder, shape):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        g = matrix(*shape, dtype=dtype, seed=shape[0], rank=max(1, min(shape) // 8))
        check(sporder.newton_schulz(g), g)


@pytest.mark.parametrize("coefficients,steps", [(MUON, 1), (MUON, 2), (MUON, 9),
                                                ((1.5, -0.5, 0.0), 12),
                                                ((1.875, -1.25, 0.375), 7),
                                                ((2.0, 0.0, 0.0), 3), ((1.0, 0.0, -0.5), 2)])
def test_coefficients_and_steps(sporder, coefficients, steps):
    for shape in ((60, 90), (300, 200)):
        g = matrix(*shape, seed=steps)
        got = sporder.newton_schulz(g, steps=steps, coefficients=coefficients)
        check(got, g, steps, coefficients)


@pytest.mark.parametrize("shape", [(1, 3, 4), (5, 40, 60), (3, 130, 70), (7, 128, 128),
                                   (2, 300, 500), (0, 4, 4)])
def test_batches(sporder, shape):
    g = matrix(*shape, seed=3)
    got = sporder.newton_schulz(g)
    assert got.shape == g.shape
    for k in range(shape[0]):
        check(got[k], g[k])
        assert torch.equal(sporder.newton_schulz(g[k]), got[k])


def test_layouts(sporder):
    wide = matrix(90, 200, seed=4)
    part = wide[:, 3:153]
    want = sporder.newton_schulz(part.contiguous())
    assert torch.equal(sporder.newton_schulz(part), want)
    assert torch.equal(sporder.newton_schulz(part.t().contiguous().t()), want)
    # The transpose goes through the same products of the same matrix.
    assert torch.equal(sporder.newton_schulz(part.t()), want.t())
    assert torch.equal(sporder.newton_schulz(part.expand(3, 90, 150)), want.expand(3, 90, 150))
    every_other = matrix(6, 40, 50, seed=5)[::2]
    assert torch.equal(sporder.newton_schulz(every_other),
                       sporder.newton_schulz(every_other.contiguous()))
    g = part.clone()
    assert sporder.newton_schulz(g, out=g) is g and torch.equal(g, want)


def test_becomes_orthogonal(sporder):
    """Thirty cubic steps bring every singular value of a matrix of condition
    below 10 to 1 within the rounding of the last steps."""
    q, _ = torch.linalg.qr(torch.randn(200, 120, dtype=torch.float64,
                                       generator=torch.Generator().manual_seed(1)))
    g = (q * torch.linspace(0.2, 1.0, 120, dtype=torch.float64)).float().cuda()
    x = sporder.newton_schulz(g, steps=30, coefficients=(1.5, -0.5, 0.0)).double()
    assert (x - q.cuda()).abs().max() < 1e-5
    assert (x.t() @ x - torch.eye(120, device="cuda", dtype=torch.float64)).abs().max() < 1e-5


def test_scale_does_not_matter(sporder):
    g = matrix(70, 150, seed=6)
    want = sporder.newton_schulz(g, eps=0.0)
    for power in (100, 30, -60, -100):
        assert torch.equal(sporder.newton_schulz(g * 2.0**power, eps=0.0), want), power


def test_zero_infinities_and_nan(sporder):
    zero = torch.zeros(50, 70, device="cuda")
    assert not sporder.newton_schulz(zero).any()
    for bad in (float("nan"), float("inf"), -float("inf")):
        g = matrix(2, 50, 70, seed=7)
        g[0, 3, 4] = bad
        got = sporder.newton_schulz(g)
        assert got[0].isnan().all()  # the formula's: every product holds it
        check(got[1], g[1])
    g = matrix(40, 60, seed=8)
    g[7], g[:, 9] = 0.0, 0.0
    got = sporder.newton_schulz(g)
    check(got, g)
    assert not got[7].any() and not got[:, 9].any()


def test_other_stream_and_graph(sporder):
    g, h = matrix(150, 260, seed=9), matrix(150, 260, seed=10)
    want = {0: sporder.newton_schulz(g), 1: sporder.newton_schulz(h)}
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = sporder.newton_schulz(g)
    s.synchronize()
    assert torch.equal(got, want[0])
    held, graph = g.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sporder.newton_schulz(held)
    for k in (1, 0, 1):
        held.copy_((g, h)[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[k])
        assert torch.equal(sporder.newton_schulz((g, h)[k]), want[k])


def test_refusals(sporder):
    g = matrix(8, 12)
    for args, kw, err in [((g.cpu(),), {}, TypeError), ((g.double(),), {}, TypeError),
                          ((g[0],), {}, ValueError), ((g[:, :0],), {}, ValueError),
                          ((g.view(1, 1, 8, 12),), {}, ValueError),
                          ((g,), {"steps": 0}, ValueError), ((g,), {"eps": -1e-7}, ValueError),
                          ((g,), {"coefficients": (1.0, 2.0)}, ValueError),
                          ((g,), {"coefficients": (16.0, 0.0, 0.0)}, ValueError),
                          ((g,), {"coefficients": (3.0, 0.0, 0.0), "steps": 3}, ValueError),
                          ((g,), {"coefficients": (3.0, 0.0, 3.0)}, ValueError),
                          ((g,), {"coefficients": (1.0, 40.0, -40.0)}, ValueError),
                          ((g,), {"coefficients": (float("nan"), 0.0, 0.0)}, ValueError),
                          ((g,), {"out": g.bfloat16()}, ValueError),
                          ((g,), {"out": g[:4]}, ValueError)]:
        with pytest.raises(err):
            sporder.newton_schulz(*args, **kw)
