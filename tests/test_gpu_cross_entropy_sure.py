"""Losses of sure rows, whose lse is many times larger than they are.

The logits are exact: row i of x is the i-th unit vector and w holds integers, so
z[i][v] = w[v][i].  A row has a target at `base`, one rival `gap` below (or above) it
and every other class 120 below the larger, whose exponential is 0 in 32 bits.  The sum
of exponentials is then 1 + e^-gap of two terms.  With u = 2^-24:

- e^-gap: its argument times log2 e is rounded twice, (2 gap) u of the value, and the
  exponential within two steps, 4 u: (2 gap + 4) u e^-gap.
- The sum is rounded once, u (1 + e^-gap) <= 2 u, which a logarithm near 1 passes on, and
  is itself within two steps of its value, 4 u of it.
- The difference of the logits is exact, one addition rounds the loss: u of it.

So a loss is within 2 u + (2 gap + 10) u of itself, whatever lse is.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# Every form of the loss: of few rows, in one pass over few classes, in tiles (of few and of
# more rows).
FORMS = [(F32, 40, 300), (BF16, 30, 300), (F32, 100, 47), (F32, 101, 47), (BF16, 300, 47),
         (F32, 129, 1000), (F16, 64, 70_000), (BF16, 256, 999)]


def sure_rows(rows, classes, dtype, seed=0):
    """x, w, targets, and by row: the target's logit less the rival's."""
    g = torch.Generator().manual_seed(seed)
    base = torch.tensor([30, 60, 100])[torch.arange(rows) % 3]
    gap = torch.arange(rows) // 3 % 17 - 1  # the rival above the target first
    target = torch.randint(0, classes, (rows,), generator=g)
    rival = (target + 1 + torch.randint(0, classes - 1, (rows,), generator=g)) % classes
    z = (base - 120.0)[:, None].expand(rows, classes).clone()
    i = torch.arange(rows)
    z[i, rival] = (base - gap).float()
    z[i, target] = base.float()
    return (torch.eye(rows).to(dtype).cuda(), z.t().contiguous().to(dtype).cuda(), target.cuda(),
            rival.cuda(), gap.double().cuda())


@pytest.mark.parametrize("dtype, rows, classes", FORMS)
def test_losses_of_sure_rows(sporder, dtype, rows, classes):
    print(f"[sure] {dtype} {rows} {classes}", flush=True)
    x, w, t, _, gap = sure_rows(rows, classes, dtype)
    loss, lse, sums = sporder.linear_cross_entropy(x, w, t)
    want = torch.nn.functional.softplus(-gap, threshold=100.0)
    tol = 2 * U + (2 * gap.abs() + 10) * U * want
    assert ((loss.double() - want).abs() <= tol).all()
    assert abs(float(sums[0]) - float(loss.double().sum())) <= 2 * U * float(want.sum())
