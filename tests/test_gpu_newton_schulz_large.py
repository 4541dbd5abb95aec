"""Newton-Schulz at the sizes where its products take the large tiles: whole
turns of them, a last row of tiles that is half empty, remainders that are
split over four and over eight waves, and batches.  Checked against the
iteration in 64 bits with the bounds of test_gpu_newton_schulz, which hold at
every size; both iterations are computed on the device."""

import pytest
import torch

from test_gpu_newton_schulz import MUON, R

pytestmark = pytest.mark.gpu


def iterate(g, dtype, steps=5, coefficients=MUON, eps=1e-7):
    x = g.to(dtype)
    if x.shape[0] > x.shape[1]:
        return iterate(g.t(), dtype, steps, coefficients, eps).t()
    a, b, c = coefficients
    x = (x / (x.double().norm() + eps).to(dtype)).contiguous()
    for _ in range(steps):
        gram = x @ x.t().contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def check(got, g):
    assert got.shape == g.shape and got.dtype == g.dtype
    exact = iterate(g, torch.float64)
    off = (got.double() - exact).norm()
    plain = (iterate(g, torch.float32).double() - exact).norm()
    # One wrong block of 32 x 32 is off by some sqrt(2 * 1024 / m) of the norm's sqrt(m).
    assert off <= 4 * plain + (2.0**-20 + R[g.dtype]) * exact.norm(), (float(off), float(plain))


def matrix(*shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rank = max(1, min(shape[-2:]) // 8)
    x = torch.randn(*shape[:-1], rank, device="cuda", generator=gen)
    y = torch.randn(*shape[:-2], rank, shape[-1], device="cuda", generator=gen)
    x = torch.matmul(x, y) + 0.5 * torch.randn(*shape, device="cuda", generator=gen)
    return (1e-3 * x).to(dtype)


# Tiles of 256 x 128 of X (updates) and, on and above the diagonal, of A:
#   (2049, 2049)  153 and 81: updates by tile, the last row of tiles half empty
#   (1500, 2500)  120 and 42: all split; (2500, 1500) the same transposed
#   (2300, 2432)  171 and 90: updates by tile, whole rows of tiles
#   (3000, 3000)  288 and 156: updates of 256 and a remainder of 32, eight waves a tile
#   (4000, 4100)  528 and 272: remainders of 16, the second on the diagonal's corner
#   (3100, 4200)  429 and 169: 173 past a turn, not split, the last rows half empty
#   (3000, 3600)  348 and 156: a remainder of 92, four waves a tile
#   (4100, 2900)  396 and 144, of the transpose
@pytest.mark.parametrize("shape,dtype", [
    ((2049, 2049), torch.float32), ((1500, 2500), torch.bfloat16), ((2500, 1500), torch.float16),
    ((2300, 2432), torch.bfloat16), ((3000, 3000), torch.float32), ((4000, 4100), torch.float32),
    ((3100, 4200), torch.float16), ((3000, 3600), torch.bfloat16), ((4100, 2900), torch.float32)])
def test_large(sporder, shape, dtype):
    print(f"[newton_schulz] {shape} {dtype}", flush=True)
    g = matrix(*shape, dtype=dtype, seed=shape[0])
    got = sporder.newton_schulz(g)
    check(got, g)
    assert torch.equal(sporder.newton_schulz(g), got)


@pytest.mark.parametrize("shape,dtype", [((16, 512, 512), torch.float32),
                                         ((40, 400, 300), torch.bfloat16),
                                         ((3, 1300, 1900), torch.float32)])
def test_large_batches(sporder, shape, dtype):
    """128 tiles or more over the batch: by tile where one matrix alone is split."""
    print(f"[newton_schulz] {shape} {dtype}", flush=True)
    g = matrix(*shape, dtype=dtype, seed=shape[0])
    got = sporder.newton_schulz(g)
    for k in range(shape[0]):
        check(got[k], g[k])
