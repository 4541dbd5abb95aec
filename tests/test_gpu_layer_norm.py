"""Layer norm and its gradients against the formula in 64 bits.

Bounds.  u = 2^-24 is half a unit of a 32-bit result, r the same of the output
type.  A row's sum has at most 64 additions in a lane, 6 across a wave and 8
across waves, or, past what a workgroup's registers hold, dim / 1024 in a
thread, 6 and 16: n = 78 + dim / 1024 additions, an error of at most n u times
the sum of magnitudes.  The terms below follow from that and one u for each
operation after it.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
R = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}


def depth(dim):
    return 78 + dim / 1024


def inputs(rows, dim, dtype, wtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=g)

    x = (normal(rows, dim) * normal(rows, 1).exp() + normal(rows, 1)).to(dtype)
    return x, normal(rows, dim).to(dtype), (1 + 0.2 * normal(dim)).to(wtype), normal(dim).to(wtype)


def check_forward(got, x, weight, bias, eps):
    y, mean, rstd = got
    dtype, dim, n = x.dtype, x.shape[-1], depth(x.shape[-1])
    xd = x.double()
    w = torch.ones(dim, device=x.device).double() if weight is None else weight.double()
    b = torch.zeros(dim, device=x.device).double() if bias is None else bias.double()
    m = xd.mean(-1, keepdim=True)
    c = xd - m
    var = (c * c).mean(-1, keepdim=True)
    rs = (var + eps).rsqrt()
    h = c * rs
    dm = (n + 2) * U * xd.abs().mean(-1, keepdim=True)
    assert mean.dtype == rstd.dtype == torch.float32 and mean.shape == x.shape[:-1] == rstd.shape
    assert ((mean.double()[..., None] - m).abs() <= dm + 1e-45).all()
    # A mean off by dm adds dm^2 to the variance.
    drel = ((n + 4) * U + dm * dm * rs * rs) / 2 + 3 * U
    assert ((rstd.double()[..., None] - rs).abs() <= drel * rs).all()
    ref = h * w + b
    tol = (w.abs() * (rs * dm + h.abs() * (drel + 4 * U)) * (1 + 1e-3)
           + 2 * U * (ref.abs() + b.abs()) + R[dtype] * ref.abs() * 1.01 + TINY[dtype])
    assert y.dtype == dtype and y.shape == x.shape
    bad = (y.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float((y.double() - ref).abs().max()))


def check_backward(got, grad, x, mean, rstd, weight, rows_depth=None):
    """Against the formula with the given mean and rstd, as inputs."""
    dx, dw, db = got
    dim, n = x.shape[-1], depth(x.shape[-1]) + 4
    x2, g2 = x.reshape(-1, dim).double(), grad.reshape(-1, dim).double()
    m, rs = mean.reshape(-1, 1).double(), rstd.reshape(-1, 1).double()
    w = torch.ones(dim, device=x.device).double() if weight is None else weight.double()
    h, gw = (x2 - m) * rs, g2 * w
    m1, m2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    ref = (gw - m1 - h * m2) * rs
    err = rs * (4 * U * gw.abs() + (n + 4) * U * gw.abs().mean(1, keepdim=True)
                + (n + 8) * U * h.abs() * (gw * h).abs().mean(1, keepdim=True)
                + 4 * U * (m1.abs() + (h * m2).abs()))
    tol = err * 1.01 + R[x.dtype] * ref.abs() * 1.01 + TINY[x.dtype]
    assert dx.dtype == x.dtype and dx.shape == x.shape
    bad = (dx.reshape(-1, dim).double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float((dx.reshape(-1, dim).double() - ref).abs().max()))
    # Column sums: any order of r rows has at most r additions.
    wtype = torch.float32 if weight is None else weight.dtype
    k = min(x2.shape[0], 200 + x2.shape[0] / 64) + 6
    for got_w, terms in ((dw, g2 * h), (db, g2)):
        assert got_w.dtype == wtype and got_w.shape == (dim,)
        ref = terms.sum(0)
        tol = k * U * terms.abs().sum(0) * 1.01 + R[wtype] * ref.abs() * 1.01 + TINY[wtype]
        assert ((got_w.double() - ref).abs() <= tol).all()


# Every lane-group width, both sides of each, odd and half-vector lengths, and
# rows past the registers of a workgroup in each direction.
DIMS = [1, 2, 3, 31, 32, 33, 47, 64, 100, 127, 128, 129, 132, 256, 257, 500, 512, 516, 1000, 1024,
        1028, 1030, 2048, 2049, 4092, 4096, 4097, 8192, 8193, 8196, 16384, 16388, 16385, 32768,
        32770, 40000]


@pytest.mark.parametrize("dim", DIMS)
def test_forward_and_backward(sporder, dim):
    for i, (dtype, wtype) in enumerate([(torch.float32, torch.float32),
                                        (torch.bfloat16, torch.float32),
                                        (torch.bfloat16, torch.bfloat16),
                                        (torch.float16, torch.float16)]):
        for rows in (1, 37) if i else (1, 2, 37, 300):
            x, g, w, b = inputs(rows, dim, dtype, wtype, seed=dim)
            got = sporder.layer_norm(x, w, b, eps=1e-5)
            check_forward(got, x, w, b, 1e-5)
            grads = sporder.layer_norm_grad(g, x, got[1], got[2], w)
            check_backward(grads, g, x, got[1], got[2], w)


@pytest.mark.parametrize("dim", [8, 48, 100, 128, 513, 1024, 4096, 20000])
def test_many_rows(sporder, dim):
    rows = min(200_000, 16_000_000 // dim) | 1
    for dtype in (torch.float32, torch.bfloat16):
        x, g, w, b = inputs(rows, dim, dtype, torch.float32, seed=dim)
        got = sporder.layer_norm(x, w, b, eps=1e-5)
        check_forward(got, x, w, b, 1e-5)
        grads = sporder.layer_norm_grad(g, x, got[1], got[2], w)
        check_backward(grads, g, x, got[1], got[2], w)
        again = sporder.layer_norm_grad(g, x, got[1], got[2], w)
        assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dim", [5, 64, 1000, 4096])
def test_without_weight_or_bias(sporder, dim):
    x, g, w, b = inputs(70, dim, torch.float32, torch.float32)
    for weight, bias in ((None, None), (w, None), (None, b)):
        got = sporder.layer_norm(x, weight, bias, eps=1e-3)
        check_forward(got, x, weight, bias, 1e-3)
        check_backward(sporder.layer_norm_grad(g, x, got[1], got[2], weight), g, x, got[1],
                       got[2], weight)


def test_layouts(sporder):
    """Leading dimensions, row strides of every alignment, broadcast rows, a
    transposed input, unaligned bases."""
    x, g, w, b = inputs(60, 96, torch.float32, torch.float32)
    want = sporder.layer_norm(x, w, b)
    want_g = sporder.layer_norm_grad(g, x, want[1], want[2], w)
    got = sporder.layer_norm(x.view(3, 4, 5, 96), w, b)
    assert got[0].shape == (3, 4, 5, 96) and got[1].shape == (3, 4, 5)
    assert torch.equal(got[0].view(60, 96), want[0])
    for pad, at in ((1, 0), (1, 1), (2, 2), (4, 4), (4, 0), (96, 0)):
        wide, wide_g = (torch.full((60, 96 + pad), float("nan"), device="cuda") for _ in range(2))
        wide[:, at:at + 96], wide_g[:, at:at + 96] = x, g
        xs, gs = wide[:, at:at + 96], wide_g[:, at:at + 96]
        got = sporder.layer_norm(xs, w, b)
        check_forward(got, x, w, b, 1e-5)
        check_backward(sporder.layer_norm_grad(gs, xs, got[1], got[2], w), g, x, got[1], got[2], w)
    xt = x.t().contiguous().t()
    assert torch.equal(sporder.layer_norm(xt, w, b)[0], want[0])
    row = x[7]
    got = sporder.layer_norm(row.expand(9, 96), w, b)
    assert torch.equal(got[0], want[0][7].expand(9, 96))
    gx = sporder.layer_norm_grad(g[7].expand(9, 96), row.expand(9, 96), got[1], got[2], w)
    assert torch.equal(gx[0], want_g[0][7].expand(9, 96))
    assert sporder.layer_norm(row, w, b)[1].shape == ()
    y = x.clone()
    assert sporder.layer_norm(y, w, b, out=y)[0] is y and torch.equal(y, want[0])


def test_no_rows(sporder):
    x = torch.empty(0, 12, device="cuda")
    w = torch.ones(12, device="cuda", dtype=torch.float32)
    y, mean, rstd = sporder.layer_norm(x, w)
    assert y.shape == (0, 12) and mean.shape == rstd.shape == (0,)
    dx, dw, db = sporder.layer_norm_grad(x, x, mean, rstd, w)
    assert dx.shape == (0, 12) and not dw.any() and not db.any()


@pytest.mark.parametrize("dim", [6, 64, 1500, 6000])
def test_rows_of_extremes(sporder, dim):
    """A constant row, a row far from zero, infinities and NaN stay in their
    own rows."""
    x, g, w, b = inputs(12, dim, torch.float32, torch.float32)
    x[2] = 3.25
    x[3] = 0.0
    x[4] = 1e6 + x[4]
    x[6, dim // 2] = float("nan")
    x[8, 0] = float("inf")
    keep = [i for i in range(12) if i not in (6, 8)]
    y, mean, rstd = sporder.layer_norm(x, w, b)
    check_forward((y[keep], mean[keep], rstd[keep]), x[keep], w, b, 1e-5)
    assert y[6].isnan().all() and mean[6].isnan()
    assert y[8].isnan().all()
    dx, _, _ = sporder.layer_norm_grad(g, x, mean, rstd, w)
    assert dx[keep].isfinite().all() and dx[6].isnan().all()
    constant = torch.full((2, dim), 0.5, device="cuda")
    assert torch.equal(sporder.layer_norm(constant, None, b)[0], b.expand(2, dim))


def test_gradients_against_differences(sporder):
    """Directional derivatives of the formula in 64 bits, by central
    differences of step 1e-5 (their error is below 1e-8 here); the kernels'
    gradients are within 1e-5 of the sum of magnitudes."""
    x, g, w, b = inputs(23, 77, torch.float32, torch.float32, seed=5)

    def loss(x, w, b):
        m = x.mean(1, keepdim=True)
        c = x - m
        return (g.double() * (c * ((c * c).mean(1, keepdim=True) + 1e-5).rsqrt() * w + b)).sum()

    _, mean, rstd = sporder.layer_norm(x, w, b)
    grads = sporder.layer_norm_grad(g, x, mean, rstd, w)
    args = [t.double() for t in (x, w, b)]
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i, grad in enumerate(grads):
        v = torch.randn(args[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-5 * v, args[i] - 1e-5 * v
        slope = float((loss(*up) - loss(*down)) / 2e-5)
        mine = grad.double() * v
        assert abs(float(mine.sum()) - slope) <= 1e-5 * float(mine.abs().sum())


def test_other_stream_and_graph(sporder):
    x, g, w, b = inputs(500, 200, torch.float32, torch.float32)
    want = sporder.layer_norm(x, w, b)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = sporder.layer_norm(x, w, b)
        grads = sporder.layer_norm_grad(g, x, got[1], got[2], w)
    s.synchronize()
    assert torch.equal(got[0], want[0])
    graph = torch.cuda.CUDAGraph()
    xs, gs = x.clone(), g.clone()
    with torch.cuda.graph(graph):
        y, mean, rstd = sporder.layer_norm(xs, w, b)
        out = sporder.layer_norm_grad(gs, xs, mean, rstd, w)
    for k in range(3):
        xs.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = sporder.layer_norm(x * (k + 1), w, b)
        eager_g = sporder.layer_norm_grad(g, x * (k + 1), eager[1], eager[2], w)
        assert torch.equal(y, eager[0])
        assert all(torch.equal(p, q) for p, q in zip(out, eager_g))
        if k == 0:
            assert all(torch.equal(p, q) for p, q in zip(out, grads))


def test_refusals(sporder):
    x, g, w, b = inputs(4, 8, torch.float32, torch.float32)
    y, mean, rstd = sporder.layer_norm(x, w, b)
    for bad, err in [(dict(x=x.cpu()), TypeError), (dict(x=x.double()), TypeError),
                     (dict(x=x[:, :0]), ValueError), (dict(x=x[0, 0]), ValueError),
                     (dict(weight=w[:7]), ValueError), (dict(weight=w.bfloat16()), TypeError),
                     (dict(bias=b.view(2, 4)), ValueError), (dict(weight=w.cpu()), TypeError),
                     (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError),
                     (dict(out=x.bfloat16()), ValueError), (dict(out=x[:3]), ValueError),
                     (dict(out=x.t().contiguous().t()), ValueError)]:
        with pytest.raises(err):
            sporder.layer_norm(**{"x": x, "weight": w, "bias": b, **bad})
    with pytest.raises(TypeError):
        sporder.layer_norm(x.bfloat16(), w, b.bfloat16())
    for bad, err in [(dict(grad=g[:3]), ValueError), (dict(grad=g.bfloat16()), TypeError),
                     (dict(mean=mean[:3]), ValueError), (dict(rstd=rstd.double()), ValueError),
                     (dict(mean=mean.cpu()), ValueError), (dict(weight=w[:3]), ValueError),
                     (dict(x=x.cpu()), TypeError)]:
        with pytest.raises(err):
            sporder.layer_norm_grad(**{"grad": g, "x": x, "mean": mean, "rstd": rstd,
                                       "weight": w, **bad})
