"""The linear cross entropy and its gradients against the formula in 64 bits.

Bounds, with u = 2^-24, A = sum_j |x_j w_j| + |bias| of a logit and r half a step
of the output's type.

- A logit is a sum of dim products in 32 bits: (dim + 16) u A.  Where 32-bit
  operands are two 16-bit halves, a product is within 2^-21 of itself and 2^-38 of
  the rows' largest elements' product.
- lse: the largest logit's error, and a sum of positive terms: classes / 16 + 100
  additions at most one after another, and exponentials whose argument is rounded
  (|z - max| e^(z - max) < 1/2): (classes / 16 + 104) u, then u |lse|.
- g = s (p - [target]): p is off by its logit's error, 4 u and the argument's
  rounding, 2 u |z - lse|; g is rounded to 11 bits (2^-11) in the products of 16-bit
  types and 22 (2^-21) in those of 32-bit ones, and nothing is below 2^-38 of s.
- A gradient is a sum of n products in 32 bits of g and operands that are rounded
  like g's for 32-bit types (exact for 16-bit ones down to 2^-39 of their column's
  largest): n u of the terms' magnitudes, 2^-21 of them, and the errors of g times
  the operands; sums in parts add a few u.
"""

import pytest
import torch

from chunkedgreedy_amd import nn

pytestmark = pytest.mark.gpu

U = 2.0**-24
R = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def inputs(rows, dim, classes, dtype, bias=None, ignored=0.0, seed=0, sure=8.0, ids=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=g)

    w = normal(classes, dim) / dim**0.5
    t = torch.randint(0, classes, (rows,), device="cuda", generator=g)
    x = normal(rows, dim) + sure * torch.rand(rows, 1, device="cuda", generator=g) * w[t]
    b = None if bias is None else (0.3 * normal(classes)).to(bias)
    t[torch.rand(rows, device="cuda", generator=g) < ignored] = -100
    s = torch.randn(rows, device="cuda", generator=g) * 0.1
    return x.to(dtype), w.to(dtype), t.to(ids), b, s


def logits(x, w, b):
    """Logits in 64 bits and the bound on their errors."""
    xd, wd = x.double(), w.double()
    z, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    dim = x.shape[1]
    err = (dim + 20) * U * size
    if x.dtype == F32:
        err = err + 2.0**-21 * size + dim * 2.0**-38 * (
            xd.abs().amax(1)[:, None] * wd.abs().amax(1)[None, :])
    return z, err


def check_loss(got, x, w, t, b, ignore=-100):
    loss, lse, sums = got
    rows, classes = x.shape[0], w.shape[0]
    assert loss.dtype == lse.dtype == sums.dtype == F32
    assert loss.shape == lse.shape == t.shape and sums.shape == (2,)
    loss, lse, t = loss.flatten(), lse.flatten(), t.flatten()
    on = t != ignore
    assert (loss[~on] == 0).all() and (lse[~on] == 0).all()
    assert float(sums[1]) == float(on.sum())
    if on.any():
        z, err = logits(x[on], w, b)
        ref = torch.logsumexp(z, 1)
        hit = torch.arange(z.shape[0], device=z.device), t[on].long()
        tol = 1.01 * (torch.where(z.isfinite(), err, torch.zeros_like(err)).amax(1)
                      + (classes / 16 + 104) * U + 2 * U * ref.abs())
        assert ((lse[on].double() - ref).abs() <= tol).all()
        want = ref - z[hit]
        tol = tol + err[hit] + 2 * U * want.abs()
        assert ((loss[on].double() - want).abs() <= tol).all()
    total = loss.double().sum()
    assert abs(float(sums[0]) - float(total)) <= 2 * U * abs(float(total)) + 1e-30


def check_grad(got, x, w, t, b, s, lse, few, ignore=-100):
    dx, dw, db = got
    rows, dim = x.shape
    classes = w.shape[0]
    on = (t != ignore)
    z, err = logits(x, w, b)
    p = torch.exp(z - lse.double()[:, None])
    g = p.clone()
    g[torch.arange(rows, device=x.device)[on], t[on].long()] -= 1.0
    s = s.double().expand(rows)[:, None] * on[:, None]
    back = 0.0 if few else 2.0**-21 if x.dtype == F32 else 2.0**-11
    arg = (z - lse.double()[:, None]).abs().clamp(max=200.0)
    off = s.abs() * (p * (err * 1.01 + (6 + 2 * arg) * U) + (back + 4 * U) * g.abs() + (0 if few else 2.0**-37))
    g = torch.where(on[:, None], g, torch.zeros_like(g)) * s
    operand = 2.0**-21 if x.dtype == F32 and not few else 0.0

    def near(value, ref, tol, kind):
        tol = 1.02 * tol + R[kind] * ref.abs() * 1.01 + TINY[kind]
        assert value.dtype == kind and value.shape == ref.shape
        bad = (value.double() - ref).abs() > tol
        assert not bad.any(), (int(bad.sum()), float(((value.double() - ref).abs() / tol).max()))

    def product(left, left_off, right):
        n = left.shape[1]
        ref = left @ right
        tol = left_off @ right.abs() + ((n + 64) * U + operand) * (left.abs() @ right.abs())
        return ref, tol + 2.0**-38 * (left.abs().sum(1, keepdim=True) * right.abs().amax(0)[None])

    xd = torch.where(on[:, None], x, torch.zeros_like(x)).double()
    near(dx, *product(g, off, w.double()), x.dtype)
    near(dw, *product(g.t().contiguous(), off.t().contiguous(), xd), dw.dtype)
    if b is None:
        assert db is None
    else:
        near(db, g.sum(0), (off + (rows + 64) * U * g.abs()).sum(0), b.dtype)
    assert (dx[~on] == 0).all()


def both(sporder, x, w, t, b, s, ignore=-100, dtype=None):
    got = sporder.linear_cross_entropy(x, w, t, b, ignore_index=ignore)
    check_loss(got, x, w, t, b, ignore)
    grads = sporder.linear_cross_entropy_grad(s, x, w, t, got[1], b, ignore_index=ignore, dtype=dtype)
    check_grad(grads, x, w, t, b, s, got[1], False, ignore)
    return got, grads


# Both sides of tiles and stages, single rows, classes and features, and sizes that
# take each form and shape.
SIZES = [(1, 1, 1), (1, 64, 300), (2, 5, 2), (7, 64, 1000), (31, 100, 500), (33, 128, 47), (64, 65, 257),
         (65, 63, 255), (129, 200, 999), (300, 64, 128), (257, 513, 256), (255, 192, 2000), (1000, 128, 47),
         (500, 16, 3), (130, 512, 40), (700, 256, 64), (90, 96, 193), (513, 1000, 700), (64, 2048, 33),
         (1030, 320, 3001)]


@pytest.mark.parametrize("rows, dim, classes", SIZES)
@pytest.mark.parametrize("dtype, bias, ids", [(F32, F32, torch.int64), (BF16, None, torch.int32),
                                              (F16, F16, torch.int64), (BF16, F32, torch.int64)])
def test_sizes(sporder, rows, dim, classes, dtype, bias, ids):
    x, w, t, b, s = inputs(rows, dim, classes, dtype, bias, 0.2, seed=rows + dim, ids=ids)
    both(sporder, x, w, t, b, s)


@pytest.mark.parametrize("classes", [1, 2, 16, 17, 33, 49, 65, 97, 129, 192])
@pytest.mark.parametrize("dim", [3, 16, 60, 128, 250])
def test_few_classes(sporder, classes, dim):
    """Every number of class blocks of the one-pass form, and dims that it leaves."""
    for dtype in (F32, BF16):
        x, w, t, b, s = inputs(333, dim, classes, dtype, dtype, 0.1, seed=classes)
        both(sporder, x, w, t, b, s)


def test_one_pass_rounds_nothing(sporder):
    """The one-pass form's 32-bit products: the bounds without any 16-bit rounding."""
    for dtype in (F32, BF16):
        x, w, t, b, s = inputs(5000, 100, 47, dtype, F32, 0.1)
        loss, lse, _ = sporder.linear_cross_entropy(x, w, t, b)
        grads = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, dtype=F32)
        check_grad(grads, x, w, t, b, s, lse, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_tiles(sporder, dtype):
    """Enough tiles for the large shape in all three products, an odd rest each way."""
    x, w, t, b, s = inputs(4100, 576, 4500, dtype, dtype, 0.1)
    both(sporder, x, w, t, b, s)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pieces_of_the_classes(sporder, dtype):
    """More logits than the scratch of one piece holds (512 MB in one order)."""
    rows, classes = 70_000, 5001 if dtype == BF16 else 2501
    x, w, t, b, s = inputs(rows, 64, classes, dtype, F32, 0.05)
    loss, lse, sums = sporder.linear_cross_entropy(x, w, t, b)
    dx, dw, db = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b)
    some = torch.arange(0, rows, 997, device="cuda")
    check_loss((loss[some], lse[some], torch.stack([loss[some].sum(), (t[some] != -100).sum().float()])),
               x[some], w, t[some], b)
    # dx by row; dw and db of all rows against 64 bits, in blocks.
    only = torch.zeros_like(s)
    only[some] = s[some]
    part = sporder.linear_cross_entropy_grad(only, x, w, t, lse, b)
    check_grad((dx[some], part[1], part[2]), x[some], w, t[some], b, s[some], lse[some], False)
    ref, size = torch.zeros(classes, 64, device="cuda", dtype=torch.float64), 0.0
    for i in range(0, rows, 10_000):
        z, _ = logits(x[i:i + 10_000], w, b)
        g = torch.exp(z - lse[i:i + 10_000].double()[:, None])
        on = t[i:i + 10_000] != -100
        g[torch.arange(g.shape[0], device="cuda")[on], t[i:i + 10_000][on]] -= 1.0
        g = torch.where(on[:, None], g, torch.zeros_like(g)) * s[i:i + 10_000].double()[:, None]
        ref += g.t().contiguous() @ x[i:i + 10_000].double()
        size = size + g.abs().t().contiguous() @ x[i:i + 10_000].double().abs()
    back = 2.0**-21 if dtype == F32 else 2.0**-11
    # Logits of |z| < 30 with sums of 64: errors of some 100 u in g's exponent.
    tol = (back * 2 + 200 * U + 1200 * U) * size + R[dtype] * ref.abs() * 1.01
    assert ((dw.double() - ref).abs() <= tol).all()


def test_many_rows_of_few_classes(sporder):
    """Long sums over the rows: every workgroup takes several tiles."""
    x, w, t, b, s = inputs(200_003, 40, 7, F32, F32, 0.3)
    both(sporder, x, w, t, b, s)


def test_long_list(sporder):
    """Past 65,536 rows the list counts its blocks first; sums over rows in parts."""
    x, w, t, b, s = inputs(70_001, 24, 260, BF16, None, 0.5)
    both(sporder, x, w, t, b, s)


@pytest.mark.parametrize("rows, dim, classes", [(300, 64, 47), (300, 96, 1000), (40, 640, 300)])
def test_layouts(sporder, rows, dim, classes):
    """Gaps between rows, odd strides and bases, other strides, more dimensions."""
    for dtype in (F32, BF16):
        x, w, t, b, s = inputs(rows, dim + 8, classes, dtype, F32, 0.1)
        for i, j in ((0, 0), (8, 0), (3, 5), (0, 1)):
            xs, ws = x[:, i:i + dim], w[:, j:j + dim]
            both(sporder, xs, ws, t, b, s)
        xs, ws = x[:, :dim].contiguous(), w[:, :dim].contiguous()
        want, grads = both(sporder, xs, ws, t, b, s)
        turned = sporder.linear_cross_entropy(xs.t().contiguous().t(), ws.t().contiguous().t(), t, b)
        assert all(torch.equal(p, q) for p, q in zip(want, turned))
        three = sporder.linear_cross_entropy(xs.view(2, rows // 2, dim), ws, t.view(2, rows // 2), b)
        assert torch.equal(three[0].flatten(), want[0])
        dx, dw, db = sporder.linear_cross_entropy_grad(
            s.view(2, rows // 2), xs.view(2, rows // 2, dim), ws, t.view(2, rows // 2), three[1], b)
        assert dx.shape == (2, rows // 2, dim)
        assert torch.equal(dx.view(rows, dim), grads[0]) and torch.equal(dw, grads[1])
        every = torch.stack([t, t], 1)[:, 0]
        assert torch.equal(sporder.linear_cross_entropy(xs, ws, every, b)[0], want[0])


@pytest.mark.parametrize("classes, dim", [(47, 128), (1000, 128), (5000, 64)])
def test_ignored_rows_are_not_read(sporder, classes, dim):
    """NaN and infinities in rows that count nothing change nothing."""
    for dtype in (F32, BF16):
        x, w, t, b, s = inputs(700, dim, classes, dtype, F32, 0.4)
        want, grads = both(sporder, x, w, t, b, s)
        bad = x.clone()
        bad[t == -100] = float("nan")
        bad[(t == -100).nonzero()[0]] = float("inf")
        got = sporder.linear_cross_entropy(bad, w, t, b)
        again = sporder.linear_cross_entropy_grad(s, bad, w, t, got[1], b)
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("classes, dim", [(47, 128), (1000, 64)])
def test_every_row_ignored_and_no_rows(sporder, classes, dim):
    x, w, t, b, s = inputs(300, dim, classes, BF16, F32)
    t[:] = -100
    loss, lse, sums = sporder.linear_cross_entropy(x, w, t, b)
    assert (loss == 0).all() and (lse == 0).all() and sums.tolist() == [0.0, 0.0]
    for grad in sporder.linear_cross_entropy_grad(s, x, w, t, lse, b):
        assert (grad == 0).all()
    loss, lse, sums = sporder.linear_cross_entropy(x[:0], w, t[:0], b)
    assert loss.shape == (0,) and sums.tolist() == [0.0, 0.0]
    dx, dw, db = sporder.linear_cross_entropy_grad(s[:0], x[:0], w, t[:0], lse, b)
    assert dx.shape == (0, dim) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("classes, dim", [(47, 128), (1000, 64)])
def test_targets_that_are_no_class(sporder, classes, dim):
    """NaN in the loss, nothing in the gradients; another ignore_index."""
    x, w, t, b, s = inputs(300, dim, classes, F32, F32)
    want = sporder.linear_cross_entropy(x, w, t, b)
    out = t.clone()
    out[5], out[77], out[200] = classes, -1, -100
    loss, lse, sums = sporder.linear_cross_entropy(x, w, out, b, ignore_index=-1)
    wrong = torch.zeros(300, dtype=torch.bool, device="cuda")
    wrong[[5, 200]] = True
    assert loss[wrong].isnan().all() and lse[wrong].isnan().all()
    assert float(loss[77]) == 0.0 and sums[0].isnan() and float(sums[1]) == 299.0
    keep = ~wrong
    keep[77] = False
    assert torch.equal(loss[keep], want[0][keep])
    grads = sporder.linear_cross_entropy_grad(s, x, w, out, lse, b, ignore_index=-1)
    masked = torch.where(keep, t, torch.full_like(t, -100))
    want = sporder.linear_cross_entropy_grad(s, x, w, masked, lse, b)
    assert all(torch.equal(p, q) for p, q in zip(grads, want))


@pytest.mark.parametrize("classes, dim", [(40, 100), (1100, 192)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_classes_left_out_by_the_bias(sporder, classes, dim, dtype):
    """A bias of -inf: no share in lse, no gradient; of the lowest value: the same."""
    x, w, t, b, s = inputs(200, dim, classes, dtype, F32)
    out = torch.zeros(classes, dtype=torch.bool, device="cuda")
    out[::3] = True
    t = torch.where(out[t], (t + 1) % classes, t)
    t = torch.where(out[t], (t + 1) % classes, t)
    for low in (float("-inf"), torch.finfo(F32).min):
        c = torch.where(out, torch.full_like(b, low), b)
        loss, lse, _ = sporder.linear_cross_entropy(x, w, t, c)
        kept = (~out).nonzero()[:, 0]
        place = torch.cumsum((~out).long(), 0) - 1
        check_loss((loss, lse, torch.stack([loss.sum(), torch.full_like(loss[0], 200.0)])), x, w[kept],
                   place[t], b[kept])
        dx, dw, db = sporder.linear_cross_entropy_grad(s, x, w, t, lse, c, dtype=F32)
        assert (dw[out] == 0).all() and (db[out] == 0).all()
        check_grad((dx, dw[kept], db[kept]), x, w[kept], place[t], b[kept], s, lse, False)
    t[:] = 0
    c = torch.full_like(b, float("-inf"))
    loss, lse, _ = sporder.linear_cross_entropy(x, w, t, c)
    assert (lse == float("-inf")).all() and loss.isnan().all()


@pytest.mark.parametrize("classes, dim", [(40, 100), (1100, 192)])
def test_scales_of_rows(sporder, classes, dim):
    """Scales far apart, zero, negative, large: each row's dx keeps its own accuracy."""
    for dtype in (F32, BF16, F16):
        x, w, t, b, s = inputs(260, dim, classes, dtype, F32)
        lse = sporder.linear_cross_entropy(x, w, t, b)[1]
        powers = torch.randint(-18, 9, (260,), device="cuda")
        s = s.sign() * 2.0**powers * (1 + torch.rand(260, device="cuda"))
        s[3] = 0.0
        got = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, dtype=F32)
        check_grad(got, x, w, t, b, s, lse, False)
        zero = sporder.linear_cross_entropy_grad(torch.zeros_like(s), x, w, t, lse, b)
        assert all((v == 0).all() for v in zero)
        one = sporder.linear_cross_entropy_grad(torch.tensor(0.37, device="cuda"), x, w, t, lse, b)
        same = sporder.linear_cross_entropy_grad(torch.full_like(s, 0.37), x, w, t, lse, b)
        wide = sporder.linear_cross_entropy_grad(torch.tensor(0.37, device="cuda").expand(260), x, w, t, lse, b)
        assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(one, same, wide))


def test_graded_features(sporder):
    """Features and classes of very different sizes, and rows far below others."""
    x, w, t, b, s = inputs(300, 128, 900, F32, None)
    size = 10.0 ** torch.linspace(-5, 2, 128, device="cuda")
    both(sporder, x * size, w / size, t, b, s)
    both(sporder, x * 1e-20, w, t, b, s)
    both(sporder, x, w * 10.0 ** torch.linspace(-30, 0, 900, device="cuda")[:, None], t, b, s)


@pytest.mark.parametrize("classes, dim", [(40, 100), (1100, 192)])
def test_sure_and_extreme_logits(sporder, classes, dim):
    for dtype in (F32, BF16):
        x, w, t, b, s = inputs(200, dim, classes, dtype, F32, sure=60.0)
        both(sporder, x, w, t, b, s)
        both(sporder, x * 30, w, t, b, s)
        x[7, 3] = float("nan")
        x[9, 1] = float("inf")
        loss, lse, _ = sporder.linear_cross_entropy(x, w, t, b)
        rest = torch.ones(200, dtype=torch.bool, device="cuda")
        rest[[7, 9]] = False
        assert loss[7].isnan() and not loss[9].isfinite()
        assert loss[rest].isfinite().all() and lse[rest].isfinite().all()


def test_weight_gradient_in_32_bits(sporder):
    for classes in (47, 1000):
        x, w, t, b, s = inputs(500, 64, classes, BF16, BF16, 0.1)
        got, grads = both(sporder, x, w, t, b, s, dtype=F32)
        assert grads[1].dtype == F32 and grads[2].dtype == BF16


@pytest.mark.parametrize("classes, dim", [(20, 30), (400, 48)])
def test_gradients_against_differences(sporder, classes, dim):
    x, w, t, b, s = inputs(50, dim, classes, F32, F32, 0.1)

    def total(x, w, b):
        z = x @ w.t() + b
        on = t != -100
        return (s.double() * on * (torch.logsumexp(z, 1) - z.gather(1, t.clamp_min(0)[:, None])[:, 0])).sum()

    lse = sporder.linear_cross_entropy(x, w, t, b)[1]
    grads = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b)
    args = [v.double() for v in (x, w, b)]
    gen = torch.Generator(device="cuda").manual_seed(3)
    for i, grad in enumerate(grads):
        v = torch.randn(args[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-5 * v, args[i] - 1e-5 * v
        slope = float((total(*up) - total(*down)) / 2e-5)
        mine = grad.double() * v
        # Differences are off by 1e-10 relative, the gradients by a few 1e-6.
        assert abs(float(mine.sum()) - slope) <= 1e-5 * float(mine.abs().sum())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("classes, dim", [(20, 30), (400, 48)])
def test_autograd(sporder, reduction, classes, dim):
    x, w, t, b, s = inputs(60, dim, classes, F32, F32, 0.2)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    loss = nn.linear_cross_entropy(leaves[0].view(2, 30, dim), leaves[1], t.view(2, 30), leaves[2],
                                   reduction=reduction)
    (loss * s.view(2, 30) if reduction == "none" else loss * 1.7).sum().backward()
    ref = [v.double().requires_grad_() for v in (x, w, b)]
    want = torch.nn.functional.cross_entropy(ref[0] @ ref[1].t() + ref[2], t, reduction=reduction)
    (want * s if reduction == "none" else want * 1.7).sum().backward()
    assert (loss.flatten().double() - want.flatten()).abs().max() <= 1e-5 * want.abs().max()
    for p, q in zip(leaves, ref):
        # Logits of |z| < 30: relative errors of some 1e-6 in p, sums of signed terms.
        assert (p.grad.double() - q.grad).abs().max() <= 1e-5 * q.grad.abs().max()
    only = x.clone().requires_grad_()
    nn.linear_cross_entropy(only, w, t).backward()
    assert only.grad.isfinite().all()
    with pytest.raises(ValueError):
        nn.linear_cross_entropy(x, w, t, reduction="max")


@pytest.mark.parametrize("rows, classes, dim", [(900, 47, 100), (500, 1500, 96), (20, 700, 64)])
def test_other_stream_and_graph(sporder, rows, classes, dim):
    x, w, t, b, s = inputs(rows, dim, classes, BF16, F32, 0.2)

    def run(x, t):
        loss, lse, sums = sporder.linear_cross_entropy(x, w, t, b)
        return (loss, lse, sums, *sporder.linear_cross_entropy_grad(s, x, w, t, lse, b))

    want = run(x, t)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = run(x, t)
    stream.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    xs, ts = x.clone(), t.clone()
    with torch.cuda.graph(graph):
        out = run(xs, ts)
    for k in range(3):
        xs.copy_(x * (k + 1) / 2)
        ts.copy_(torch.roll(t, k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, run(x * (k + 1) / 2, torch.roll(t, k))))


def test_refusals(sporder):
    x, w, t, b, s = inputs(12, 8, 20, F32, F32)
    lse = sporder.linear_cross_entropy(x, w, t, b)[1]
    base = {"x": x, "weight": w, "targets": t, "bias": b}
    bads = [(dict(x=x.cpu()), TypeError), (dict(x=x.double()), TypeError), (dict(x=x[:, :0]), ValueError),
            (dict(weight=w.half()), TypeError), (dict(weight=w[:, :7]), ValueError),
            (dict(weight=w[0]), ValueError), (dict(weight=w[:0]), ValueError), (dict(targets=t[:5]), ValueError),
            (dict(targets=t.float()), TypeError), (dict(targets=t.cpu()), TypeError),
            (dict(bias=b[:5]), ValueError), (dict(bias=b.half()), TypeError), (dict(bias=b.cpu()), TypeError),
            (dict(ignore_index=2**63), ValueError)]
    for bad, err in bads:
        with pytest.raises(err):
            sporder.linear_cross_entropy(**{**base, **bad})
        with pytest.raises(err):
            sporder.linear_cross_entropy_grad(s, lse=lse, **{**base, **bad})
    for bad, err in [(dict(grad=s[:5]), ValueError), (dict(grad=s.double()), TypeError),
                     (dict(grad=s.cpu()), TypeError), (dict(lse=lse[:5]), ValueError),
                     (dict(lse=lse.half()), TypeError), (dict(dtype=BF16), ValueError)]:
        with pytest.raises(err):
            sporder.linear_cross_entropy_grad(**{"grad": s, "lse": lse, **base, **bad})
    with pytest.raises(ValueError):
        wide = torch.zeros(1, 65537, device="cuda")
        sporder.linear_cross_entropy(wide, wide, t[:1])


@pytest.mark.parametrize("dim", [8, 9, 15, 33, 64, 99, 130, 255, 257, 300, 388, 500, 512])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_few_classes_by_lengths(sporder, dim, dtype):
    """The loss's one-pass form over rows that end inside its accesses, at odd
    places and strides, with each number of class blocks."""
    for classes in (1, 16, 30, 47, 64, 90, 128, 172, 192):
        for rows in (1, 17, 150):
            x, w, t, b, _ = inputs(rows, dim + 3, classes, dtype, dtype, 0.1, seed=dim + classes)
            xs, ws = x[:, 1:dim + 1], w[:, 2:dim + 2]
            check_loss(sporder.linear_cross_entropy(xs, ws, t, b), xs, ws, t, b)


@pytest.mark.parametrize("dtype, dim", [(F32, 40), (BF16, 40), (F32, 260), (F32, 500)])
def test_few_classes_of_many_rows(sporder, dtype, dim):
    """More rows than the workgroups' waves take at a time; rows that count nothing,
    and a first row that counts and holds no numbers, touch no other."""
    rows = 140_003 if dim < 100 else 70_003
    x, w, t, b, _ = inputs(rows, dim, 12, dtype, F32, 0.3, seed=3)
    t[0] = 1
    want = sporder.linear_cross_entropy(x, w, t, b)
    check_loss(want, x, w, t, b)
    x[0] = float("nan")
    loss, lse, sums = sporder.linear_cross_entropy(x, w, t, b)
    assert loss[0].isnan() and lse[0].isnan() and sums[0].isnan()
    assert torch.equal(loss[1:], want[0][1:]) and torch.equal(lse[1:], want[1][1:])


def test_few_classes_past_the_tiles_rows(sporder):
    """2^23 + 77 rows, which only the one-pass form takes."""
    rows = 2**23 + 77
    x, w, t, b, s = inputs(rows, 8, 3, BF16, F32, 0.1, seed=4)
    loss, lse, sums = sporder.linear_cross_entropy(x, w, t, b)
    dx, dw, db = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b)
    some = torch.cat([torch.arange(0, rows, 99_991, device="cuda"),
                      torch.arange(rows - 90, rows, device="cuda")])
    check_loss((loss[some], lse[some], torch.stack([loss[some].sum(), (t[some] != -100).sum().float()])),
               x[some], w, t[some], b)
    assert float(sums[1]) == float((t != -100).sum())
    p = torch.softmax(x.double() @ w.double().t() + b.double(), 1)
    on = t != -100
    p[torch.arange(rows, device="cuda")[on], t[on]] -= 1.0
    g = p * (s * on).double()[:, None]
    # 2^23 terms of |g| <= |s|; the sums' parts add up to some 2^-24 of the magnitudes a step.
    size = g.abs().sum(0)
    assert ((db.double() - g.sum(0)).abs() <= (rows / 256 / 512 + 600) * U * size).all()
    want = g.t().contiguous() @ x.double()
    size = g.abs().t().contiguous() @ x.double().abs()
    assert ((dw.double() - want).abs() <= (2.0**-8 * want.abs() + 2.0**-11 * size)).all()
    got = dx[some].double() - (g[some] @ w.double())
    bound = 2.0**-8 * (g[some] @ w.double()).abs() + 2.0**-11 * (g[some].abs() @ w.double().abs())
    assert (got.abs() <= bound + 2.0**-126).all()


@pytest.mark.parametrize("dtype, rows", [(F32, 1), (F32, 29), (F32, 64), (BF16, 20), (F16, 32)])
def test_few_rows_that_count_nothing_are_not_read(sporder, dtype, rows):
    """The form of few rows: NaN and infinities in ignored rows and in rows whose target is
    no class change nothing."""
    x, w, t, b, s = inputs(rows + 3, 200, 777, dtype, F32, 0.3, seed=rows)
    x, t, s = x[:rows], t[:rows], s[:rows]
    t[0] = 5
    want, grads = both(sporder, x, w, t, b, s)
    bad = x.clone()
    bad[t == -100] = float("nan")
    if (t == -100).any():
        bad[(t == -100).nonzero()[0]] = float("inf")
    got = sporder.linear_cross_entropy(bad, w, t, b)
    again = sporder.linear_cross_entropy_grad(s, bad, w, t, got[1], b)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    if rows > 1:
        out = t.clone()
        out[1] = 777
        got = sporder.linear_cross_entropy(bad, w, out, b)
        assert got[0][1].isnan() and got[0][0] == want[0][0]
        dx, dw, db = sporder.linear_cross_entropy_grad(s, bad, w, out, got[1], b)
        assert (dx[1] == 0).all() and dw.isfinite().all() and db.isfinite().all()


def test_calls_at_once_on_two_streams(sporder):
    """Each form on two streams at a time, each call with scratch of its own."""
    cases = [(F32, 20, 96, 3000), (BF16, 900, 96, 3000), (F32, 5000, 96, 40), (BF16, 5000, 300, 100)]
    for dtype, rows, dim, classes in cases:
        sets = [inputs(rows, dim, classes, dtype, F32, 0.1, seed=k) for k in range(2)]
        want = [both(sporder, *v) for v in sets]
        streams = [torch.cuda.Stream() for _ in range(2)]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for _ in range(4):
            for k, stream in enumerate(streams):
                x, w, t, b, s = sets[k]
                with torch.cuda.stream(stream):
                    loss = sporder.linear_cross_entropy(x, w, t, b)
                    got[k].append((loss, sporder.linear_cross_entropy_grad(s, x, w, t, loss[1], b)))
        torch.cuda.synchronize()
        for k in range(2):
            for loss, grads in got[k]:
                assert all(torch.equal(p, q) for p, q in zip(loss, want[k][0]))
                assert all(torch.equal(p, q) for p, q in zip(grads, want[k][1]))


@pytest.mark.parametrize("rows", [1, 32, 50])
@pytest.mark.parametrize("dim", [1024, 1003])
def test_few_rows_of_large_weights(sporder, rows, dim):
    """16-bit weights on either side of 2^25 elements, which few rows take in two forms."""
    for classes in (34_001, 3001):
        x, w, t, b, s = inputs(rows, dim, classes, BF16, BF16, 0.1, seed=rows + dim)
        both(sporder, x, w, t, b, s)
