"""The linear cross entropy's forms one by one: rows that count nothing beside weights that are
no numbers, and the gradients of few classes under the bounds of the form that makes them.

Bounds as in test_gpu_cross_entropy.py.  Where tiles are shared by the workgroup, all products
are of 32 bits: nothing but sums is rounded.  Where each wave has its own, logits and dx are
products of 22 bits whatever the type, in units of w's rows and columns and x's rows (g's
smaller half in steps of 2^-24 of 2^13: nothing below 2^-38 of the scale), dw of 32 bits.
"""

import pytest
import torch

from test_gpu_cross_entropy import BF16, F16, F32, R, TINY, U, check_grad, inputs, logits

pytestmark = pytest.mark.gpu

# Few rows; one pass with a tile for each wave; with tiles shared by the workgroup (16 and 32
# bits, odd and even lengths); tiles.
FORMS = [(F32, 40, 64, 300), (BF16, 20, 64, 300), (F32, 300, 100, 47), (BF16, 300, 64, 16),
         (F32, 300, 101, 47), (BF16, 300, 101, 47), (F32, 300, 256, 60), (BF16, 300, 40, 192),
         (F16, 300, 320, 10), (F32, 300, 7, 47), (F32, 300, 64, 1000), (BF16, 300, 64, 1000)]


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype, rows, dim, classes", FORMS)
def test_rows_that_count_nothing_beside_weights_that_are_no_numbers(sporder, dtype, rows, dim, classes, bad):
    """Their gradients are 0 whatever weights hold."""
    print(f"[forms] {dtype} {rows} {dim} {classes} {bad}", flush=True)
    x, w, t, b, s = inputs(rows, dim, classes, dtype, F32, 0.4, seed=dim)
    t[0], t[1], t[rows - 1] = -100, classes, -100
    w[classes // 2, dim // 3] = bad
    w[0] = -bad
    loss, lse, _ = sporder.linear_cross_entropy(x, w, t, b)
    off = (t < 0) | (t >= classes)
    assert (loss[t == -100] == 0).all() and (lse[t == -100] == 0).all() and loss[1].isnan()
    for given in (None, loss):
        dx = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, loss=given)[0]
        assert (dx[off] == 0).all()


@pytest.mark.parametrize("dim, classes", [(101, 47), (256, 60), (9, 3), (63, 192), (127, 100), (383, 16)])
def test_tiles_shared_by_the_workgroup_round_nothing(sporder, dim, classes):
    """Rows of odd length, and more of w than leaves room for a tile for each wave: the
    bounds without any 16-bit rounding."""
    for dtype in (F32, BF16):
        print(f"[forms] shared {dtype} {dim} {classes}", flush=True)
        x, w, t, b, s = inputs(3001, dim, classes, dtype, F32, 0.1, seed=dim)
        loss, lse, _ = sporder.linear_cross_entropy(x, w, t, b)
        for given in (None, loss):
            grads = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, dtype=F32, loss=given)
            check_grad(grads, x, w, t, b, s, lse, True)


@pytest.mark.parametrize("dim, classes", [(100, 47), (64, 64), (128, 48), (192, 30), (8, 2), (60, 16)])
def test_tiles_of_a_wave_keep_22_bits(sporder, dim, classes):
    for dtype in (F32, BF16, F16):
        print(f"[forms] of a wave {dtype} {dim} {classes}", flush=True)
        x, w, t, b, s = inputs(3001, dim, classes, dtype, F32, 0.1, seed=dim)
        lse = sporder.linear_cross_entropy(x, w, t, b)[1]
        dx, dw, db = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, dtype=F32)
        on = t != -100
        z, _ = logits(x, w, b)
        xd, wd = x.double(), w.double()
        size = xd.abs() @ wd.abs().t() + b.double().abs()
        err = (dim + 20) * U * size + 2.0**-21 * size + dim * 2.0**-38 * (
            xd.abs().amax(1)[:, None] * wd.abs().amax(1)[None, :])
        away = (z - lse.double()[:, None]).abs().clamp(max=200.0)
        p = torch.exp(z - lse.double()[:, None])
        g = p.clone()
        g[torch.arange(3001, device="cuda")[on], t[on]] -= 1.0
        scale = (s.double() * on)[:, None]
        off = scale.abs() * (p * (1.01 * err + (6 + 2 * away) * U) + 4 * U * g.abs())
        g = torch.where(on[:, None], g, torch.zeros_like(g)) * scale

        def near(value, ref, tol):
            tol = 1.02 * tol + R[value.dtype] * ref.abs() * 1.01 + TINY[value.dtype]
            assert ((value.double() - ref).abs() <= tol).all()

        kept = off + 2.0**-21 * g.abs() + 2.0**-38 * scale.abs()
        tol = kept @ wd.abs() + ((classes + 64) * U + 2.0**-21) * (g.abs() @ wd.abs())
        near(dx, g @ wd, tol + 2.0**-38 * g.abs().sum(1, keepdim=True) * wd.abs().amax(0)[None])
        left, xd = g.t().contiguous(), torch.where(on[:, None], xd, torch.zeros_like(xd))
        near(dw, left @ xd, off.t().contiguous() @ xd.abs() + (3001 + 64) * U * (left.abs() @ xd.abs()))
        near(db, g.sum(0), (off + (3001 + 64) * U * g.abs()).sum(0))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_scale_of_all_rows_does_not_touch_gs_bits(sporder, dtype):
    """Tiles of 16-bit types.  Undecided rows over C classes have a g of 1 / C - 1 for their
    target, which 11 bits hold to 2^-12, whatever the one scale of all rows is: chosen here so
    that g times its mantissa would lie halfway between two values of 11 bits above 1, 2^-11
    from each.  Row i's x is the i-th unit vector: column i of w's gradient is g."""
    rows = 200
    print(f"[forms] one scale {dtype}", flush=True)
    x = torch.eye(rows, device="cuda").to(dtype)
    for classes in (211, 500, 1000, 2001, 5003):
        w = torch.zeros(classes, rows, device="cuda", dtype=dtype)
        t = torch.arange(rows, device="cuda") * 7 % classes
        lse = sporder.linear_cross_entropy(x, w, t)[1]
        hit = 1.0 - 1.0 / classes
        for power, sign in ((0, 1), (-9, 1), (5, -1)):
            scale = sign * 2.0**power * (1.0 + 2.0**-11 - 2.0**-20) / hit
            s = torch.full((rows,), scale, device="cuda")
            s[3:5] *= -1  # a scale's sign is no bit of g
            for grad in (s, torch.tensor(scale, device="cuda")):
                dw = sporder.linear_cross_entropy_grad(grad, x, w, t, lse, dtype=F32)[1]
                g = dw[t, torch.arange(rows, device="cuda")].double() / grad.double()
                # Beside the 11 bits: lse's rounding and the scale's, u of 9 and of g.
                assert ((g + hit).abs() <= 2.0**-12 + 16 * U).all()
