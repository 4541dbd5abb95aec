"""The training operators where sizes change their course: few tokens of a
large table, tensors of more than 2^31 elements, rows of unaligned 16- and
32-bit elements at the lengths where their accesses change; and what the
differentiable forms refuse."""

import pytest
import torch

from test_gpu_layer_norm import check_backward, check_forward, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sporder():
    from chunkedgreedy_amd import sporder
    return sporder


def whole(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-4, 5, shape, device="cuda", generator=g).to(dtype)


# Whole numbers from -4 to 4, at most 8192 to a row: every order of the sums
# gives the same 32-bit result, rounded once.
@pytest.mark.parametrize("count", [0, 1, 2, 63, 64, 65, 300, 1024, 1025, 2500, 4096, 4097, 8192])
@pytest.mark.parametrize("kind", ["spread", "one", "two", "outside"])
def test_few_tokens_of_a_large_table(sporder, kind, count):
    rows = 300_000
    g = torch.Generator(device="cuda").manual_seed(count)
    tok = torch.randint(0, rows, (count,), device="cuda", generator=g)
    if kind == "one":
        tok.fill_(rows - 1)
    elif kind == "two":
        tok = torch.where(tok % 3 == 0, 7, 299_998)
    elif kind == "outside":
        tok = torch.where(tok % 3 == 0, -1, torch.where(tok % 3 == 1, rows, tok % 50))
    for dim, dtype, out in [(64, torch.float32, torch.float32), (64, torch.bfloat16, torch.bfloat16),
                            (60, torch.float16, torch.float32), (57, torch.bfloat16, torch.float32)]:
        grad = whole((count, dim), dtype, count + dim)
        keep = (tok >= 0) & (tok < rows) & (tok != 7)
        want = torch.zeros(rows, dim, device="cuda", dtype=torch.float64)
        want.index_add_(0, tok[keep], grad[keep].double())
        got = torch.full((rows, dim), float("nan"), device="cuda", dtype=out)
        sporder.embedding_grad(grad, tok.int(), rows, scale=0.5, padding_idx=7, dtype=out, out=got)
        assert torch.equal(got, (0.5 * want).to(out))


def test_lookup_past_31_bits(sporder):
    rows, dim = 2_200_000, 1024 # 2.25e9 elements
    table = torch.zeros(rows, dim, device="cuda", dtype=torch.bfloat16)
    last = whole((5, dim), torch.bfloat16, 1)
    table[-5:] = last
    tok = torch.tensor([rows - 1, 0, rows - 5, rows - 1, 2**21], device="cuda")
    assert torch.equal(sporder.embedding(table, tok, scale=2.0), 2.0 * table[tok])
    del table
    for count in (5, 100_000): # a workgroup per token, and sorted tiles
        far = tok.repeat(count // 5)
        grad = whole((count, dim), torch.bfloat16, 2)
        if count > 5:
            grad[5:] = 0 # the sums stay whole numbers below 2^8, exact in 16 bits
        out = sporder.embedding_grad(grad, far, rows)
        want = torch.zeros(5, dim, device="cuda")
        want.index_add_(0, (far[:5] - (rows - 5)).clamp(min=0) * (far[:5] >= rows - 5),
                        grad[:5].float() * (far[:5] >= rows - 5)[:, None])
        assert torch.equal(out[-5:].float(), want)
        assert torch.equal(out[0], grad[1]) and torch.equal(out[2**21], grad[4])
        out[-5:] = 0
        out[0] = 0
        out[2**21] = 0
        assert not torch.any(out.view(torch.int16).view(-1, 1024).any(1)).item()
        del out
    wide = torch.zeros(2_200_000, dim, device="cuda", dtype=torch.bfloat16)
    out = sporder.embedding(last, torch.full((2_200_000,), 3, device="cuda"), out=wide)
    assert torch.equal(out[-1], last[3]) and torch.equal(out[2**21 + 7], last[3])


def test_layer_norm_past_31_bits(sporder):
    rows, dim = 2**21 + 5, 1024
    x = torch.zeros(rows, dim, device="cuda", dtype=torch.bfloat16)
    x[:8], x[-8:] = whole((8, dim), torch.bfloat16, 3), whole((8, dim), torch.bfloat16, 4)
    x[8:-8] = whole((1, dim), torch.bfloat16, 5)
    y, mean, rstd = sporder.layer_norm(x)
    dy = whole((1, dim), torch.bfloat16, 6).expand(rows, dim) # stride 0
    dx, dw, db = sporder.layer_norm_grad(dy, x, mean, rstd)
    for part in (slice(0, 8), slice(2**20, 2**20 + 8), slice(rows - 8, rows)):
        y8, mean8, rstd8 = sporder.layer_norm(x[part])
        dx8, _, _ = sporder.layer_norm_grad(dy[part], x[part], mean8, rstd8)
        assert torch.equal(y[part], y8) and torch.equal(mean[part], mean8)
        assert torch.equal(rstd[part], rstd8) and torch.equal(dx[part], dx8)
    assert torch.equal(db, dy[0].float() * rows) # whole numbers below 2^24: exact


@pytest.mark.parametrize("dim", [3, 5, 7, 9, 31, 63, 127, 129, 257, 513, 1025, 2049, 4095, 4097,
                                 8191, 8193, 16383, 16385, 32767])
def test_layer_norm_of_unaligned_rows(sporder, dim):
    """Rows a stride apart, off every vector, with NaN between them."""
    rows = 37
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x, dy, w, b = inputs(rows, dim, dtype, torch.float32, seed=dim)
        apart = torch.full((2, rows * (dim + 1) + 1), float("nan"), device="cuda").to(dtype)
        xs, dys = (flat[1:].view(rows, dim + 1)[:, :dim] for flat in apart)
        xs.copy_(x)
        dys.copy_(dy)
        got = sporder.layer_norm(xs, w, b, eps=1e-5)
        check_forward(got, x, w, b, 1e-5)
        check_backward(sporder.layer_norm_grad(dys, xs, got[1], got[2], w), dy, x, got[1], got[2], w)


def test_what_the_differentiable_forms_refuse(sporder):
    from chunkedgreedy_amd import nn
    table = torch.randn(10, 4, device="cuda", requires_grad=True)
    tok = torch.tensor([1, 2], device="cuda")
    for pad in (-1, 10):
        with pytest.raises(ValueError):
            sporder.embedding_grad(torch.randn(2, 4, device="cuda"), tok, 10, padding_idx=pad)
    with pytest.raises(ValueError):
        sporder.newton_schulz(torch.randn(4, 4, device="cuda"), steps=2**32 + 1)
    for y in (nn.embedding(table, tok), nn.layer_norm(table)):
        first, = torch.autograd.grad(y.pow(2).sum(), table, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), table)
    with pytest.raises(ValueError):
        nn.Muon([torch.randn(4, device="cuda", requires_grad=True)])
