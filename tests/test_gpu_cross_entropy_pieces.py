"""The gradients of the linear cross entropy over rows that are cut into pieces.

Bounds as in test_gpu_cross_entropy.py, with a gradient by w or bias of n rows summed in parts
of at most 2^20 rows, by 16 rows a matrix instruction or, for the bias, by 32 a wave and then
workgroup by workgroup: at most n / 16 + 100 additions one after another, u of the terms'
magnitudes each.
"""

import pytest
import torch

from test_gpu_cross_entropy import BF16, F16, F32, R, TINY, U, inputs, logits

pytestmark = pytest.mark.gpu


def check_in_blocks(got, x, w, t, b, s, lse, block):
    dx, dw, db = got
    rows, dim = x.shape
    back = 2.0**-21 if x.dtype == F32 else 2.0**-11
    operand = 2.0**-21 if x.dtype == F32 else 0.0
    zeros = lambda *n: torch.zeros(*n, device=x.device, dtype=torch.float64)  # noqa: E731
    ref_w, off_w = zeros(*w.shape), zeros(*w.shape)
    ref_b, off_b = zeros(w.shape[0]), zeros(w.shape[0])
    wd, most = w.double(), x.abs().amax(0).double()

    def near(value, ref, tol):
        tol = 1.02 * tol + R[value.dtype] * ref.abs() * 1.01 + TINY[value.dtype]
        bad = (value.double() - ref).abs() > tol
        assert not bad.any(), (int(bad.sum()), float(((value.double() - ref).abs() / tol).max()))

    for i in range(0, rows, block):
        xi, ti, li = x[i:i + block], t[i:i + block], lse[i:i + block].double()[:, None]
        on = ti != -100
        z, err = logits(xi, w, b)
        p = torch.exp(z - li)
        g = p.clone()
        g[torch.arange(g.shape[0], device=x.device)[on], ti[on]] -= 1.0
        scale = (s[i:i + block].double() * on)[:, None]
        arg = (z - li).abs().clamp(max=200.0)
        off = scale.abs() * (p * (1.01 * err + (6 + 2 * arg) * U) + (back + 4 * U) * g.abs() + 2.0**-37)
        g = torch.where(on[:, None], g, torch.zeros_like(g)) * scale
        n = w.shape[0]
        tol = off @ wd.abs() + ((n + 64) * U + operand) * (g.abs() @ wd.abs())
        tol = tol + 2.0**-38 * g.abs().sum(1, keepdim=True) * wd.abs().amax(0)[None]
        near(dx[i:i + block], g @ wd, tol)
        assert (dx[i:i + block][~on] == 0).all()
        xd = torch.where(on[:, None], xi, torch.zeros_like(xi)).double()
        left, left_off = g.t().contiguous(), off.t().contiguous()
        ref_w += left @ xd
        off_w += left_off @ xd.abs() + ((rows / 16 + 100) * U + operand) * (left.abs() @ xd.abs())
        off_w += 2.0**-38 * left.abs().sum(1, keepdim=True) * most[None]
        ref_b += g.sum(0)
        off_b += (off + (rows / 16 + 100) * U * g.abs()).sum(0)
    near(dw, ref_w, off_w)
    if b is not None:
        near(db, ref_b, off_b)


@pytest.mark.parametrize("dtype, rows, dim, classes, bias, ignored", [
    (F32, 140_003, 24, 900, F32, 0.05),   # two pieces of the rows
    (F32, 140_003, 20, 2001, F32, 0.1),   # and two of the classes
    (BF16, 530_001, 16, 300, BF16, 0.0),
    (BF16, 1_050_001, 33, 211, F32, 0.6),  # the second piece's rows count nothing
    (F16, 2_100_007, 9, 230, None, 0.1),  # three pieces
    (F32, 16_500, 8192, 210, F32, 0.1),   # cut for their length
    (BF16, 33_001, 8192, 250, None, 0.2)])
def test_pieces_of_the_rows(sporder, dtype, rows, dim, classes, bias, ignored):
    print(f"[pieces of the rows] {dtype} {rows} {dim} {classes}", flush=True)
    x, w, t, b, s = inputs(rows, dim, classes, dtype, bias, ignored, seed=rows + classes)
    lse = sporder.linear_cross_entropy(x, w, t, b)[1]
    for kind in {dtype, F32}:
        got = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, dtype=kind)
        assert got[1].dtype == kind
        check_in_blocks(got, x, w, t, b, s, lse, max(1000, 20_000_000 // (classes + dim)))
        again = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, dtype=kind)
        assert all(p is q is None or torch.equal(p, q) for p, q in zip(got, again))


def test_pieces_without_rows_that_count(sporder):
    """No row counts, or only the last ones: zeros, and what those rows alone give."""
    print("[pieces of the rows] few count", flush=True)
    x, w, t, b, s = inputs(140_003, 16, 850, F32, F32, 0.0, seed=1)
    none = torch.full_like(t, -100)
    lse = torch.zeros_like(s)
    for g in sporder.linear_cross_entropy_grad(s, x, w, none, lse, b):
        assert (g == 0).all()
    none[-70:] = t[-70:]
    lse = sporder.linear_cross_entropy(x, w, none, b)[1]
    dx, dw, db = sporder.linear_cross_entropy_grad(s, x, w, none, lse, b)
    check_in_blocks((dx, dw, db), x, w, none, b, s, lse, 70_000)
    assert (dx[:-70] == 0).all() and (dx[-70:] != 0).any()


def test_pieces_of_the_rows_captured(sporder):
    print("[pieces of the rows] captured", flush=True)
    x, w, t, b, s = inputs(140_003, 12, 800, F32, F32, 0.1, seed=2)

    def run(x, t):
        lse = sporder.linear_cross_entropy(x, w, t, b)[1]
        return sporder.linear_cross_entropy_grad(s, x, w, t, lse, b)

    run(x, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    xs, ts = x.clone(), t.clone()
    with torch.cuda.graph(graph):
        out = run(xs, ts)
    for k in range(3):
        xs.copy_(x * (k + 1) / 2)
        ts.copy_(torch.roll(t, k))
        graph.replay()
        torch.cuda.synchronize()
        want = run(x * (k + 1) / 2, torch.roll(t, k))
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_rows_that_only_the_loss_takes_in_one_pass(sporder):
    """2^23 + 77 rows over 172 classes, whose loss is the one-pass form's and whose gradients
    are the tiles': the forward call takes them, and so does the backward pass."""
    rows, dim, classes = 2**23 + 77, 129, 172
    print(f"[pieces of the rows] {rows} {dim} {classes}", flush=True)
    x, w, t, b, s = inputs(rows, dim, classes, BF16, F32, 0.1, seed=9)
    lse = sporder.linear_cross_entropy(x, w, t, b)[1]
    got = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, dtype=F32)
    check_in_blocks(got, x, w, t, b, s, lse, 200_000)


def test_rows_refused_by_the_forward_call(sporder):
    """More rows than the gradients take: the forward call says so."""
    x = torch.zeros(1, 8, device="cuda").expand(2**23, 8)
    t = torch.zeros((), device="cuda", dtype=torch.int64).expand(2**23)
    for classes, dim in ((193, 8), (100, 7)):
        w = torch.zeros(classes, dim, device="cuda")
        with pytest.raises(ValueError, match="rows"):
            sporder.linear_cross_entropy(x[:, :dim], w, t)
