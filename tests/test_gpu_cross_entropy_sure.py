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

The gradients: row i's x is the i-th unit vector, so column i of w's gradient is g[i], in 32
bits where it is asked for.  The target's g is e^-loss - 1 = -p and the rival's
p = e^-gap / (1 + e^-gap):

- The target's: the loss is off by 2 u + (2 gap + 10) u of it, as above; below a loss of 1/2
  the exponential's difference from 1 by two steps, 4 u of it, above that e^-loss is off by
  (2 loss + 4) u of itself, 3 u at most; the row's scale rounds it, and its
  products keep 22 or 11 bits of it.
- The rival's: exp(z - lse) of a difference off by lse's rounding, u |lse|, and by the
  argument's, (2 gap + 4) u; its rounding as the target's.
- Of g times 2^13 the smaller half of 32-bit types has steps of 2^-24, half of which is 2^-38
  of the scale (16-bit types' steps are as small where 11 bits of g do not count for more).
"""

import pytest
import torch

from chunkedgreedy_amd import nn

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


# What g keeps in its products, whatever the form: 22 bits of 32-bit types, 11 of 16-bit ones.
BACK = {F32: 2.0**-21, BF16: 2.0**-11, F16: 2.0**-11}


@pytest.mark.parametrize("dtype, rows, classes", FORMS)
def test_gradients_of_sure_rows(sporder, dtype, rows, classes):
    print(f"[sure gradients] {dtype} {rows} {classes}", flush=True)
    x, w, t, rival, gap = sure_rows(rows, classes, dtype)
    loss, lse, _ = sporder.linear_cross_entropy(x, w, t)
    scale = torch.full((rows,), 1.5, device="cuda")
    dx, dw, _ = sporder.linear_cross_entropy_grad(scale, x, w, t, lse, dtype=F32, loss=loss)
    g = dw.double() / 1.5  # [class][row]
    rows_of = torch.arange(rows, device="cuda")
    p = 1.0 / (1.0 + torch.exp(gap))
    want = torch.nn.functional.softplus(-gap, threshold=100.0)
    back = BACK[dtype] + 4 * U
    tol = 2 * U + (2 * gap.abs() + 10) * U * want + (4 * U + back) * p + 2.0**-38 + 3 * U * (want >= 0.5)
    assert ((g[t, rows_of] + p).abs() <= 1.01 * tol).all()
    tol = ((lse.double().abs() + 2 * gap.abs() + 8) * U + back) * p + 2.0**-38
    assert ((g[rival, rows_of] - p).abs() <= 1.01 * tol).all()
    g[t, rows_of] = 0.0
    g[rival, rows_of] = 0.0
    assert (g == 0).all()


@pytest.mark.parametrize("rows, classes", [(40, 300), (100, 47), (101, 47), (129, 1000)])
def test_autograd_of_sure_rows(sporder, rows, classes):
    """The differentiable form takes the loss by itself, and the losses that it returns may
    be written to."""
    print(f"[sure autograd] {rows} {classes}", flush=True)
    x, w, t, _, _ = sure_rows(rows, classes, F32)
    loss, lse, _ = sporder.linear_cross_entropy(x, w, t)
    scale = torch.rand(rows, device="cuda")
    want = sporder.linear_cross_entropy_grad(scale, x, w, t, lse, loss=loss)
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    out = nn.linear_cross_entropy(*leaves, t, reduction="none")
    assert torch.equal(out, loss)
    out *= scale
    out.sum().backward()
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[1].grad, want[1])
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    nn.linear_cross_entropy(*leaves, t).backward()
    mean = torch.ones((), device="cuda") / rows
    want = sporder.linear_cross_entropy_grad(mean, x, w, t, lse, loss=loss)
    assert torch.equal(leaves[1].grad, want[1])


@pytest.mark.parametrize("dtype, rows, classes", [(F32, 40, 300), (F32, 100, 47), (F32, 101, 47),
                                                  (BF16, 256, 999)])
def test_given_losses_of_any_row(sporder, dtype, rows, classes):
    """Losses that are 0, infinite and NaN, of ignored rows and of targets that are no class;
    strided losses; a loss of other values is refused by its shape, type and place."""
    print(f"[given losses] {dtype} {rows} {classes}", flush=True)
    x, w, t, _, _ = sure_rows(rows, classes, dtype)
    bias = torch.zeros(classes, device="cuda")
    bias[t[4]] = float("-inf")  # rows of this target: an infinite loss, g of the target -1
    t[5], t[6] = -100, classes
    x[7] = float("nan")
    loss, lse, _ = sporder.linear_cross_entropy(x, w, t, bias)
    assert loss[4] == float("inf") and loss[7].isnan() and loss[6].isnan() and loss[5] == 0
    keep = ~loss.isnan()
    scale = keep.float()
    t = torch.where(t == t[7], torch.full_like(t, -100), t)  # its class has a gradient of NaN
    x[7] = 0.0
    t[7] = -100
    with_loss = sporder.linear_cross_entropy_grad(scale, x, w, t, lse, bias, dtype=F32, loss=loss)
    without = sporder.linear_cross_entropy_grad(scale, x, w, t, lse, bias, dtype=F32)
    for p, q in zip(with_loss, without):
        assert p.isfinite().all()
        # lse is at most 121: its rounding is all that they differ by.
        assert ((p.double() - q.double()).abs() <= 128 * 121 * U * 2 + 2.0**-8 * q.double().abs()).all()
    assert (with_loss[0][5] == 0).all() and (with_loss[0][6] == 0).all()
    apart = torch.stack([loss, loss], 1)[:, 0]
    again = sporder.linear_cross_entropy_grad(scale, x, w, t, lse, bias, dtype=F32, loss=apart)
    assert all(torch.equal(p, q) for p, q in zip(with_loss, again))
    for bad, err in ((loss[:5], ValueError), (loss.half(), TypeError), (loss.cpu(), TypeError)):
        with pytest.raises(err):
            sporder.linear_cross_entropy_grad(scale, x, w, t, lse, bias, loss=bad)


def test_entry_without_losses(sporder):
    """The C entry that takes no losses gives what the other gives for NULL."""
    from chunkedgreedy_amd import _lib

    x, w, t, _, _ = sure_rows(129, 1000, F32)
    lse = sporder.linear_cross_entropy(x, w, t)[1]
    one = torch.ones(1, device="cuda")
    want = sporder.linear_cross_entropy_grad(one, x, w, t, lse)
    lib = _lib.load()
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    sizes = (129, x.data_ptr(), 129, w.data_ptr())
    size = lib.sporder_linear_cross_entropy_grad_work_bytes(_lib.TYPE_F32, 129, 129, 1000, *sizes)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    assert lib.sporder_linear_cross_entropy_grad(
        torch.cuda.current_stream().cuda_stream, _lib.TYPE_F32, 129, 129, 1000, 0, one.data_ptr(), *sizes,
        _lib.TYPE_F32, 0, 64, t.data_ptr(), -100, lse.data_ptr(), 129, dx.data_ptr(), _lib.TYPE_F32, 129,
        dw.data_ptr(), 0, work.data_ptr(), size) == _lib.OK
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
