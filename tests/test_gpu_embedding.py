"""Row lookup and the table gradient.

The lookup is one product and one rounding per element: compared bit for bit.
The gradient is compared bit for bit on whole numbers, whose sums are exact in
32 bits in any order, and within n u of the sum of magnitudes (n summands, u =
2^-24, and one rounding to the output type) on real ones.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
R = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ids(kind, count, rows, seed=0):
    g = gen(seed)
    u = torch.rand(count, device="cuda", generator=g, dtype=torch.float64)
    if kind == "uniform":
        return (u * rows).long().clamp_(max=rows - 1)
    if kind == "zipf":
        rank = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
        return torch.randperm(rows, device="cuda", generator=g)[rank]
    if kind == "one":
        return torch.full((count,), rows - 1, device="cuda", dtype=torch.int64)
    if kind == "two":
        return torch.where(u < 0.3, 0, rows // 2)
    if kind == "sorted":
        return (u * rows).long().clamp_(max=rows - 1).sort().values
    if kind == "close":  # a few neighbouring rows take everything
        return rows // 3 + (u * min(8, rows - rows // 3)).long()
    if kind == "outside":  # a third below zero or past the table
        return (u * rows * 1.5).long() - rows // 4
    raise ValueError(kind)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [1, 3, 4, 8, 32, 33, 100, 128, 260, 1000, 1024, 2050, 8192])
def test_lookup(sporder, dim, dtype):
    rows = 777
    table = torch.randn(rows, dim, device="cuda", generator=gen(dim)).to(dtype)
    for count in (0, 1, 5, 300):
        for scale in (1.0, 11.313708):
            tok = ids("uniform", count, rows, seed=count)
            want = (table[tok].float() * torch.tensor(scale, dtype=torch.float32)).to(dtype)
            for t in (tok, tok.int()):
                got = sporder.embedding(table, t, scale=scale)
                assert got.dtype == dtype and torch.equal(got, want)


def test_lookup_layouts(sporder):
    base = torch.randn(50, 70, device="cuda", generator=gen(1))
    tok = ids("uniform", 24, 50).view(2, 3, 4)
    for table in (base[:, 1:65], base[:, 4:68], base[::2, :64], base.t()[:64, :50].t(),
                  base[3].expand(50, 70)):
        t = tok % table.shape[0]
        got = sporder.embedding(table, t, scale=0.5)
        assert got.shape == (2, 3, 4, table.shape[1])
        assert torch.equal(got, table[t] * 0.5)
    out = torch.empty(24, 70, device="cuda")
    assert sporder.embedding(base, tok.view(24)[::1], out=out) is out
    assert torch.equal(sporder.embedding(base, tok.view(24)[::2]), base[tok.view(24)[::2]])


def test_lookup_outside_the_table(sporder):
    table = torch.randn(10, 6, device="cuda")
    tok = torch.tensor([3, -1, 10, 9, 2**40, -(2**62), 0], device="cuda")
    got = sporder.embedding(table, tok)
    assert got[[1, 2, 4, 5]].isnan().all()
    assert torch.equal(got[[0, 3, 6]], table[[3, 9, 0]])


def whole_numbers(count, dim, dtype, seed):
    return torch.randint(-8, 9, (count, dim), device="cuda", generator=gen(seed)).to(dtype)


def reference(grad, tok, rows, padding=None):
    keep = (tok >= 0) & (tok < rows)
    if padding is not None:
        keep &= tok != padding
    out = torch.zeros(rows, grad.shape[1], device="cuda", dtype=torch.float64)
    return out.index_add_(0, tok[keep], grad[keep].double())


COUNTS = [0, 1, 2, 63, 64, 65, 128, 1000, 4095, 4096, 4097, 8192, 30_000]


@pytest.mark.parametrize("count", COUNTS)
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "two", "sorted", "close", "outside"])
def test_grad_whole_numbers(sporder, kind, count):
    for rows, dim in ((1, 5), (2, 64), (300, 33), (2049, 8), (20_000, 20), (300_000, 4)):
        tok = ids(kind, count, rows, seed=rows)
        grad = whole_numbers(count, dim, torch.float32, count)
        got = sporder.embedding_grad(grad, tok, rows)
        want = reference(grad, tok, rows)
        assert got.shape == (rows, dim)
        assert torch.equal(got.double(), want), (rows, dim)


@pytest.mark.parametrize("dim", [1, 4, 7, 32, 100, 128, 260, 1024, 1100, 4100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_grad_real_numbers(sporder, dim, dtype):
    rows, count = 5000, 9000
    tok = ids("zipf", count, rows, seed=dim)
    grad = torch.randn(count, dim, device="cuda", generator=gen(dim)).to(dtype)
    want = reference(grad, tok, rows, 17) * 3.0
    terms = reference(grad.abs(), tok, rows, 17) * 3.0
    n = torch.bincount(tok, minlength=rows).double()[:, None]
    for out in {dtype, torch.float32}:
        got = sporder.embedding_grad(grad, tok.int(), rows, scale=3.0, padding_idx=17, dtype=out)
        assert got.dtype == out and not got[17].any()
        tol = (n + 1) * U * terms * 1.01 + R[out] * want.abs() * 1.01 + TINY[out]
        assert ((got.double() - want).abs() <= tol).all()
        again = sporder.embedding_grad(grad, tok, rows, scale=3.0, padding_idx=17, dtype=out)
        assert torch.equal(got, again)


@pytest.mark.parametrize("kind,rows", [("zipf", 2_000_000), ("uniform", 1000), ("close", 60_000),
                                       ("one", 7), ("outside", 100_000)])
def test_grad_many_tokens(sporder, kind, rows):
    count, dim = 400_001, 12
    tok = ids(kind, count, rows, seed=3)
    grad = whole_numbers(count, dim, torch.float32, 4)
    got = sporder.embedding_grad(grad, tok, rows, padding_idx=rows // 2)
    # Sums of up to 400,001 numbers below 9 in magnitude: exact in 32 bits.
    assert torch.equal(got.double(), reference(grad, tok, rows, rows // 2))


def test_grad_layouts(sporder):
    tok = ids("zipf", 600, 40)
    wide = whole_numbers(600, 80, torch.float32, 1)
    for grad in (wide[:, 1:65], wide[:, 4:68], wide[:, :64], wide.t().contiguous().t(),
                 wide[3].expand(600, 80)):
        assert torch.equal(sporder.embedding_grad(grad, tok, 40).double(),
                           reference(grad, tok, 40))
    got = sporder.embedding_grad(wide.view(20, 30, 80), tok.view(20, 30), 40)
    assert torch.equal(got.double(), reference(wide, tok, 40))
    out = torch.full((40, 80), float("nan"), device="cuda")
    assert sporder.embedding_grad(wide, tok, 40, out=out) is out
    assert torch.equal(out, got)


def test_grad_infinities_and_nan_stay_in_their_rows(sporder):
    tok = torch.tensor([3, 4, 3, 5, 6, 9], device="cuda")
    grad = torch.ones(6, 40, device="cuda")
    grad[1, 7], grad[3, 8], grad[4] = float("nan"), float("inf"), float("nan")
    got = sporder.embedding_grad(grad, tok, 12, padding_idx=6)
    want = torch.zeros(12, 40, device="cuda")
    want[3], want[4], want[5], want[9] = 2.0, 1.0, 1.0, 1.0
    want[4, 7], want[5, 8] = float("nan"), float("inf")
    assert torch.equal(got.nan_to_num(7.5), want.nan_to_num(7.5))


def test_grad_against_differences(sporder):
    """The lookup is linear: sum(grad * (E(table + v) - E(table - v))) / 2
    equals sum(dtable * v), in whole numbers exactly."""
    rows, dim, count = 90, 24, 700
    tok = ids("zipf", count, rows)
    grad = whole_numbers(count, dim, torch.float32, 2)
    table, v = (whole_numbers(rows, dim, torch.float32, s) for s in (3, 4))
    slope = (grad * (sporder.embedding(table + v, tok, scale=2.0)
                     - sporder.embedding(table - v, tok, scale=2.0))).double().sum() / 2
    got = sporder.embedding_grad(grad, tok, rows, scale=2.0)
    assert float((got * v).double().sum()) == float(slope)


def test_other_stream_and_graph(sporder):
    rows, dim, count = 3000, 48, 5000
    tok, other = ids("zipf", count, rows, 1), ids("uniform", count, rows, 2)
    grad = whole_numbers(count, dim, torch.float32, 5)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = sporder.embedding_grad(grad, tok, rows)
    s.synchronize()
    assert torch.equal(got.double(), reference(grad, tok, rows))
    held, graph = tok.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sporder.embedding_grad(grad, held, rows)
        back = sporder.embedding(out, held)
    for t in (tok, other, tok):
        held.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = reference(grad, t, rows)
        assert torch.equal(out.double(), want) and torch.equal(back.double(), want[t])


def test_refusals(sporder):
    table = torch.randn(10, 4, device="cuda")
    tok = torch.tensor([1, 2], device="cuda")
    grad = torch.randn(2, 4, device="cuda")
    for args, kw, err in [((table.cpu(), tok), {}, TypeError), ((table, tok.cpu()), {}, TypeError),
                          ((table, tok.float()), {}, TypeError),
                          ((table.double(), tok), {}, TypeError),
                          ((table[0], tok), {}, ValueError), ((table[:0], tok), {}, ValueError),
                          ((table, tok), {"out": grad.bfloat16()}, ValueError),
                          ((table, tok), {"out": grad[:1]}, ValueError)]:
        with pytest.raises(err):
            sporder.embedding(*args, **kw)
    for args, kw, err in [((grad.cpu(), tok, 10), {}, TypeError),
                          ((grad, tok[:1], 10), {}, ValueError),
                          ((grad, tok.short(), 10), {}, TypeError),
                          ((grad, tok, 0), {}, ValueError), ((grad, tok, 2**31), {}, ValueError),
                          ((grad, tok, 10), {"dtype": torch.bfloat16}, ValueError),
                          ((grad, tok, 10), {"out": grad}, ValueError)]:
        with pytest.raises(err):
            sporder.embedding_grad(*args, **kw)
