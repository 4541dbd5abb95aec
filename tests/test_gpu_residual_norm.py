"""The norms around a block and their gradients against the formula in 64 bits.

Bounds.  u = 2^-24, r half a step of the output's type.  A row's sum has at most
64 additions in a lane, 6 across a wave and 8 across waves, or dim / 1024 in a
thread, 6 and 16 past the registers: at most n = 78 + dim / 1024, an error of n u
times the sum of magnitudes; each operation after it adds one u.  A sum of
squares has no cancellation, so rstd is within (n + 4) u / 2 + 3 u of itself.
"""

import pytest
import torch

from chunkedgreedy_amd import nn

pytestmark = pytest.mark.gpu

U = 2.0**-24
R = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}


def depth(dim):
    return 78 + dim / 1024


def inputs(rows, dim, dtype, wtype, gate="vector", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=g)

    t = {"x": (normal(rows, dim) * normal(rows, 1).exp()).to(dtype),
         "residual": normal(rows, dim).to(dtype), "gate": None,
         "post_weight": (1 + 0.2 * normal(dim)).to(wtype),
         "weight": (1 + 0.2 * normal(dim)).to(wtype)}
    if gate == "vector":
        t["gate"] = normal(dim).to(wtype)
    elif gate == "rows":
        t["gate"] = torch.sigmoid(normal(rows, dim)).to(dtype)
    return t, normal(rows, dim).to(dtype), normal(rows, dim).to(dtype)


def wide(t, like):
    return torch.ones((), device=like.device, dtype=torch.float64) if t is None else t.double()


def check_forward(got, t, scale, eps, post=True):
    y, h, r1, r2 = got
    x, dtype = t["x"], t["x"].dtype
    dim, n = x.shape[-1], depth(x.shape[-1])
    xd = x.double()
    res = 0.0 if t["residual"] is None else t["residual"].double()
    rel = (n + 4) * U / 2 + 3 * U
    one = ((xd * xd).mean(-1) + eps).rsqrt() if post else torch.ones_like(xd[..., 0])
    assert r1.dtype == r2.dtype == torch.float32 and r1.shape == r2.shape == x.shape[:-1]
    assert ((r1.double() - one).abs() <= rel * one).all()
    part = xd * one[..., None] * wide(t["post_weight"], x) * wide(t["gate"], x) * scale
    ref = res + part
    # Five products and a sum after post_rstd; scale itself is rounded.
    err = (rel + 7 * U) * part.abs() + U * ref.abs()
    tol = 1.01 * err + R[dtype] * ref.abs() * 1.01 + TINY[dtype]
    assert y.dtype == h.dtype == dtype and y.shape == h.shape == x.shape
    assert ((y.double() - ref).abs() <= tol).all()
    # y's errors enter h's norm: a row's mean square is off by 2 mean |y| err at most.
    square = (ref * ref).mean(-1)
    two = (square + eps).rsqrt()
    off = 1.01 * (ref.abs() * err).mean(-1) * two * two
    rel2 = rel + off
    assert ((r2.double() - two).abs() <= rel2 * two * 1.01).all()
    w2 = wide(t["weight"], x)
    ref_h = ref * two[..., None] * w2
    tol = (1.02 * (err * two[..., None] * w2.abs() + (rel2[..., None] + 3 * U) * ref_h.abs())
           + R[dtype] * ref_h.abs() * 1.01 + TINY[dtype])
    assert ((h.double() - ref_h).abs() <= tol).all()


def check_backward(got, dy, dh, t, y, r1, r2, scale, post=True):
    dx, dres, dgate, dw1, dw2 = got
    x = t["x"]
    dtype, dim, n = x.dtype, x.shape[-1], depth(x.shape[-1]) + 4
    rows = x.numel() // dim
    flat = lambda v: v.reshape(-1, dim).double()  # noqa: E731
    xd, yd = flat(x), flat(y)
    dyd = torch.zeros_like(xd) if dy is None else flat(dy)
    dhd = torch.zeros_like(xd) if dh is None else flat(dh)
    r1, r2 = r1.reshape(-1, 1).double(), r2.reshape(-1, 1).double()
    by_row = t["gate"] is not None and t["gate"].dim() == x.dim() > 1
    gate = flat(t["gate"]) if by_row else wide(t["gate"], x)
    w1, w2 = wide(t["post_weight"], x), wide(t["weight"], x)
    yhat, b = yd * r2, dhd * w2
    m1 = (b * yhat).mean(1, keepdim=True)
    e = dyd + r2 * (b - yhat * m1)
    e_err = (r2 * (4 * U * b.abs() + (n + 6) * U * yhat.abs() * (b * yhat).abs().mean(1, keepdim=True))
             + 2 * U * e.abs())

    def near(value, ref, err, kind):
        tol = 1.02 * err + R[kind] * ref.abs() * 1.01 + TINY[kind]
        assert value.dtype == kind
        bad = (value.double().reshape(ref.shape) - ref).abs() > tol
        assert not bad.any(), (int(bad.sum()), float((value.double().reshape(ref.shape) - ref).abs().max()))

    near(dres, e, e_err, dtype)
    xhat = xd * r1
    gain = scale * w1 * gate
    a = e * gain
    a_err = (e_err + 5 * U * e.abs()) * gain.abs()
    m2 = (a * xhat).mean(1, keepdim=True) if post else torch.zeros_like(r1)
    m2_err = ((n + 2) * U * (a * xhat).abs() + a_err * xhat.abs()).mean(1, keepdim=True) if post else 0.0
    ref = (a - xhat * m2) * r1
    near(dx, ref, r1 * (a_err + xhat.abs() * m2_err + 3 * U * (a.abs() + (xhat * m2).abs())), dtype)
    # Column sums: rows in a lane, then groups, waves and partial rows.
    k = min(rows, 200 + rows / 64) + 12
    kind = torch.float32
    for v in (t["post_weight"], t["weight"], None if by_row else t["gate"]):
        kind = kind if v is None else v.dtype

    def column(value, terms, errs):
        near(value, terms.sum(0), (k * U * terms.abs() + errs).sum(0), kind)

    part = scale * xhat * (e * gate if by_row else e)
    part_err = scale * xhat.abs() * (e_err + 6 * U * e.abs()) * (gate.abs() if by_row else 1.0)
    if dw1 is not None:
        column(dw1, part * (1.0 if by_row else gate), part_err * (1.0 if by_row else gate.abs()))
    if t["gate"] is not None:
        if by_row:
            near(dgate, scale * w1 * xhat * e, (scale * w1 * xhat).abs() * (e_err + 6 * U * e.abs()), dtype)
        else:
            column(dgate, part * w1, part_err * w1.abs())
    if dw2 is not None:
        column(dw2, dhd * yhat, 3 * U * (dhd * yhat).abs())


# Every lane-group width, both sides of each, odd and half-vector lengths, and
# rows past the registers of a workgroup in each direction.
DIMS = [1, 2, 3, 16, 17, 33, 64, 100, 127, 128, 129, 256, 260, 500, 513, 1000, 1024, 1025, 2048,
        2050, 4096, 4100, 8192, 8193, 16384, 16386, 20000]


def both(sporder, t, dy, dh, scale=0.5, eps=1e-5, post=True):
    y, h, r1, r2 = got = sporder.residual_norm(**t, scale=scale, eps=eps, post_norm=post)
    check_forward(got, t, scale, eps, post)
    rest = {k: t[k] for k in ("gate", "post_weight", "weight")}
    grads = sporder.residual_norm_grad(dy, dh, t["x"], y, r1, r2, **rest, scale=scale, post_norm=post)
    check_backward(grads, dy, dh, t, y, r1, r2, scale, post)
    return got, grads


@pytest.mark.parametrize("dim", DIMS)
def test_forward_and_backward(sporder, dim):
    kinds = [(torch.float32, torch.float32, "vector"), (torch.bfloat16, torch.float32, "rows"),
             (torch.float16, torch.float16, "none"), (torch.bfloat16, torch.bfloat16, "vector")]
    for i, (dtype, wtype, gate) in enumerate(kinds):
        t, dy, dh = inputs(37, dim, dtype, wtype, gate, seed=i)
        both(sporder, t, dy, dh)


@pytest.mark.parametrize("dim", [8, 100, 128, 1000, 4096, 9000])
@pytest.mark.parametrize("gate", ["none", "vector", "rows"])
def test_many_rows(sporder, dim, gate):
    t, dy, dh = inputs(300_000 // dim + 5001 // (1 + dim // 500), dim, torch.float32, torch.float32, gate)
    both(sporder, t, dy, dh, scale=1.0)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65])
def test_few_rows(sporder, rows):
    for dim in (1, 40, 512, 4096):
        t, dy, dh = inputs(rows, dim, torch.bfloat16, torch.float32, "rows")
        both(sporder, t, dy, dh)


@pytest.mark.parametrize("dim", [5, 64, 1000, 4096, 20000])
def test_parts_left_out(sporder, dim):
    t, dy, dh = inputs(41, dim, torch.float32, torch.float32, "vector")
    for missing in (["residual"], ["post_weight"], ["weight"], ["gate"],
                    ["residual", "gate", "post_weight", "weight"]):
        both(sporder, {k: None if k in missing else v for k, v in t.items()}, dy, dh)
    both(sporder, t, None, dh)
    both(sporder, t, dy, None)
    both(sporder, t, None, None)
    for gate in (None, t["gate"], torch.rand_like(t["x"])):
        both(sporder, {**t, "post_weight": None, "gate": gate}, dy, dh, post=False)


def test_layouts(sporder):
    for dim in (48, 64, 100, 1030):
        t, dy, dh = inputs(60, dim + 8, torch.bfloat16, torch.float32, "rows")
        cut = {k: v[:, 3:dim + 3] if v.dim() == 2 else v[:dim] for k, v in t.items()}
        both(sporder, cut, dy[:, 1:dim + 1], dh[:, 5:dim + 5])
        three = {k: v[:, :dim].reshape(3, 20, dim) if v.dim() == 2 else v[:dim] for k, v in t.items()}
        both(sporder, three, dy[:, :dim].reshape(3, 20, dim), dh[:, :dim].reshape(3, 20, dim))
        turned = {k: v[:, :dim].t().contiguous().t() if v.dim() == 2 else v[:dim] for k, v in t.items()}
        both(sporder, turned, dy[:, :dim], dh[:, :dim])
        one = {**cut, "x": cut["x"][:1].expand(60, dim), "gate": cut["gate"][:1].expand(60, dim)}
        both(sporder, one, dy[:, :dim], dh[:, :dim])


def test_no_rows(sporder):
    t, dy, dh = inputs(0, 12, torch.float32, torch.float32)
    y, h, r1, r2 = sporder.residual_norm(**t)
    assert y.shape == h.shape == (0, 12) and r1.shape == (0,)
    grads = sporder.residual_norm_grad(dy, dh, t["x"], y, r1, r2, t["gate"], t["post_weight"],
                                       t["weight"])
    assert grads[0].shape == (0, 12) and all((g == 0).all() for g in grads[2:])


@pytest.mark.parametrize("dim", [6, 64, 1500, 20000])
def test_rows_of_extremes(sporder, dim):
    """Rows of zeros, tiny and large values; a row of NaN stays in its row."""
    t, dy, dh = inputs(6, dim, torch.float32, torch.float32, "none")
    t["x"][0] = 0.0
    t["residual"][0] = 0.0
    t["x"][1] *= 1e-20
    t["x"][2] *= 1e15
    t["residual"][3] *= 1e15
    both(sporder, t, dy, dh, scale=1.0)
    t["x"][4] = float("nan")
    y, h, r1, r2 = sporder.residual_norm(**t)
    assert y[4].isnan().all() and h[4].isnan().all()
    assert y[[0, 1, 2, 3, 5]].isfinite().all() and h[[0, 1, 2, 3, 5]].isfinite().all()


def test_gradients_against_differences(sporder):
    """Directional derivatives of the formula in 64 bits."""
    t, dy, dh = inputs(9, 24, torch.float32, torch.float32, "vector", seed=5)

    def loss(v):
        x, res, gate, w1, w2 = v
        y = res + 0.7 * gate * w1 * x * ((x * x).mean(-1, keepdim=True) + 1e-3).rsqrt()
        h = w2 * y * ((y * y).mean(-1, keepdim=True) + 1e-3).rsqrt()
        return (y * dy.double()).sum() + (h * dh.double()).sum()

    y, h, r1, r2 = sporder.residual_norm(**t, scale=0.7, eps=1e-3)
    grads = sporder.residual_norm_grad(dy, dh, t["x"], y, r1, r2, t["gate"], t["post_weight"],
                                       t["weight"], scale=0.7)
    args = [v.double() for v in t.values()]
    gen = torch.Generator(device="cuda").manual_seed(8)
    for i, grad in enumerate(grads):
        v = torch.randn(args[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-5 * v, args[i] - 1e-5 * v
        slope = float((loss(up) - loss(down)) / 2e-5)
        mine = grad.double() * v
        # Differences are off by 1e-10 relative, the gradients by a few 1e-6.
        assert abs(float(mine.sum()) - slope) <= 1e-5 * float(mine.abs().sum())


@pytest.mark.parametrize("gate", ["none", "vector", "rows"])
def test_autograd(sporder, gate):
    t, dy, dh = inputs(30, 20, torch.float32, torch.float32, gate, seed=6)
    leaves = {k: None if v is None else v.clone().requires_grad_() for k, v in t.items()}
    y, h = nn.residual_norm(**leaves, scale=0.3, eps=1e-4)
    ((y * dy).sum() + (h * dh).sum()).backward()
    mine = {k: None if v is None else v.grad for k, v in leaves.items()}
    ref = {k: None if v is None else v.double().requires_grad_() for k, v in t.items()}
    x = ref["x"]
    u = x * ((x * x).mean(-1, keepdim=True) + 1e-4).rsqrt() * ref["post_weight"] * 0.3
    yy = ref["residual"] + (u if ref["gate"] is None else u * ref["gate"])
    hh = yy * ((yy * yy).mean(-1, keepdim=True) + 1e-4).rsqrt() * ref["weight"]
    ((yy * dy).sum() + (hh * dh).sum()).backward()
    for k, v in ref.items():
        if v is not None:
            # Sums of at most 30 terms or 20, each within some 100 u.
            assert (mine[k].double() - v.grad).abs().max() <= 2e-5 * v.grad.abs().max()
    # Only one of the outputs used; leaves that want no gradient.
    x = t["x"].clone().requires_grad_()
    nn.residual_norm(x, t["residual"], t["gate"])[1].sum().backward()
    assert x.grad.isfinite().all()
    nn.residual_norm(x, None, None)[0].sum().backward()


def test_other_stream_and_graph(sporder):
    t, dy, dh = inputs(500, 200, torch.float32, torch.float32, "vector")
    rest = {k: t[k] for k in ("gate", "post_weight", "weight")}

    def run(x):
        y, h, r1, r2 = sporder.residual_norm(**{**t, "x": x})
        return (y, h, r1, r2, *sporder.residual_norm_grad(dy, dh, x, y, r1, r2, **rest))

    want = run(t["x"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(t["x"])
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    x = t["x"].clone()
    with torch.cuda.graph(graph):
        out = run(x)
    for k in range(3):
        x.copy_(t["x"] * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, run(t["x"] * (k + 1))))


def test_refusals(sporder):
    t, dy, dh = inputs(4, 8, torch.float32, torch.float32)
    y, h, r1, r2 = sporder.residual_norm(**t)
    for bad, err in [(dict(x=t["x"].cpu()), TypeError), (dict(x=t["x"].double()), TypeError),
                     (dict(x=t["x"][:, :0]), ValueError), (dict(residual=t["x"][:3]), ValueError),
                     (dict(residual=t["x"].half()), TypeError), (dict(gate=t["gate"][:7]), ValueError),
                     (dict(gate=t["x"][:3]), ValueError), (dict(gate=t["x"].half()), TypeError),
                     (dict(weight=t["weight"].half()), TypeError), (dict(eps=-1.0), ValueError),
                     (dict(weight=t["weight"].cpu()), TypeError), (dict(eps=float("nan")), ValueError),
                     (dict(post_norm=False), ValueError)]:
        with pytest.raises(err):
            sporder.residual_norm(**{**t, **bad})
    with pytest.raises(TypeError):
        half = {**t, "x": t["x"].half(), "residual": None, "weight": t["weight"].half()}
        sporder.residual_norm(**half)
    good = {"grad_y": dy, "grad_h": dh, "x": t["x"], "y": y, "post_rstd": r1, "rstd": r2,
            "gate": t["gate"], "post_weight": t["post_weight"], "weight": t["weight"]}
    for bad, err in [(dict(grad_y=dy[:3]), ValueError), (dict(grad_h=dh.half()), TypeError),
                     (dict(y=y[:3]), ValueError), (dict(rstd=r2[:3]), ValueError),
                     (dict(post_rstd=r1.double()), ValueError), (dict(rstd=r2.cpu()), ValueError),
                     (dict(y=y.cpu()), TypeError), (dict(post_norm=False), ValueError)]:
        with pytest.raises(err):
            sporder.residual_norm_grad(**{**good, **bad})
