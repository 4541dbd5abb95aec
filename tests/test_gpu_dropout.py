"""Dropout from a counter against its definition: the generator in 64-bit host
integers, the values in 64 bits.

Bounds.  A kept element is x (1 / (1 - p)) with the factor rounded to 32 bits, the
product rounded to 32 bits, the residual added with one more rounding, and the
result rounded to its type: 3 u of the parts' magnitudes and r of the result, u =
2^-24 and r half a step of the type.
"""

import numpy as np
import pytest
import torch

from chunkedgreedy_amd import nn

pytestmark = pytest.mark.gpu

U = 2.0**-24
R = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}


def philox(block, offset, seed, plane):
    """Four words per block (numpy uint64 holding 32 bits)."""
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    c = [block & m, block >> s, np.full_like(block, offset & 0xFFFFFFFF),
         np.full_like(block, (offset >> 32) | plane << 31)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> s) ^ c[1] ^ np.uint64(k[0]), q & m, (p >> s) ^ c[3] ^ np.uint64(k[1]), p & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def random_bits(n, seed, offset, first=0):
    """The 32 bits of elements first .. first + n."""
    i = np.arange(first, first + n, dtype=np.uint64)
    out = np.zeros(n, np.uint64)
    for plane, shift in ((0, 16), (1, 0)):
        words = philox(i >> np.uint64(3), offset, seed, plane)
        word = np.choose((i % np.uint64(8) // np.uint64(2)).astype(np.int64), words)
        half = np.where(i & np.uint64(1), word >> np.uint64(16), word & np.uint64(0xFFFF))
        out |= half << np.uint64(shift)
    return out


def check(out, x, p, seed, offset, residual=None):
    keep = random_bits(x.numel(), seed, offset) >= np.uint64(round(p * 2**32))
    keep = torch.from_numpy(keep).to(x.device).view(x.shape)
    ref = torch.where(keep, x.double() / (1 - p) if p < 1 else torch.zeros_like(x).double(),
                      torch.zeros((), dtype=torch.float64, device=x.device))
    size = ref.abs()
    if residual is not None:
        ref, size = ref + residual.double(), size + residual.double().abs()
    assert out.shape == x.shape and out.dtype == x.dtype and out.is_contiguous()
    tol = 3.01 * U * size + R[x.dtype] * ref.abs() * 1.01 + TINY[x.dtype]
    assert ((out.double() - ref).abs() <= tol).all()
    if residual is None:
        assert (out[~keep] == 0).all()
    else:
        assert torch.equal(out[~keep], residual[~keep])
    return keep


SEED, OFFSET = 0xFEDCBA9876543210, 0x7123456789ABCDEF


@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (511,), (512,), (3, 5), (64, 512),
                                   (1000, 33), (3, 17, 130), (4097, 1029)])
@pytest.mark.parametrize("dtype", list(R))
def test_values(sporder, shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(shape, device="cuda", generator=g).to(dtype)
    res = torch.randn(shape, device="cuda", generator=g).to(dtype)
    check(sporder.dropout(x, 0.3, SEED, offset=OFFSET), x, 0.3, SEED, OFFSET)
    check(sporder.dropout(x, 0.1, 5, offset=2, residual=res), x, 0.1, 5, 2, res)


def test_many_elements(sporder):
    """Both sides of where a lane takes several blocks, an odd length, and the
    share that is dropped: within 6 standard deviations."""
    for n in (2**23 - 8, 2**23 + 8, 2**23 + 13):
        x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
        keep = check(sporder.dropout(x, 0.1, 3, offset=9), x, 0.1, 3, 9)
        assert abs(float((~keep).float().mean()) - 0.1) < 6 * (0.09 / n) ** 0.5


@pytest.mark.parametrize("p", [0.0, 1.0, 2.0**-32, 2.0**-33, 0.5, 2.0**-16, 1 - 2.0**-32, 0.1,
                               3 * 2.0**-17])
def test_probabilities(sporder, p):
    """The ends of the range, thresholds with and without low bits (where ties of
    the high halves decide), and rounding to steps of 2^-32."""
    x = torch.randn(300_000, device="cuda")
    keep = check(sporder.dropout(x, p, 11, offset=0), x, p, 11, 0)
    if p in (0.0, 2.0**-33):
        assert keep.all()
    if p == 1.0:
        assert not keep.any()


def test_ties_take_the_low_bits(sporder):
    """p chosen at one element's own bits: it is kept, and dropped one step above."""
    bits = random_bits(4096, 77, 5)
    x = torch.ones(4096, device="cuda")
    for i in (0, 1, 6, 7, 1003, 4095):
        t = int(bits[i])
        for step, kept in ((0, True), (1, False)):
            p = (t + step) / 2**32
            out = sporder.dropout(x, p, 77, offset=5)
            assert (float(out[i]) != 0) == kept
            check(out, x, p, 77, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_share_the_mask(sporder, dtype):
    """Gaps between rows, other strides, unaligned bases: the mask goes by the
    index in the shape."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for rows, dim in ((40, 33), (40, 64), (300, 7), (5, 1000)):
        big = torch.randn(rows, dim + 9, device="cuda", generator=g).to(dtype)
        res = torch.randn(rows, dim + 5, device="cuda", generator=g).to(dtype)[:, 2:dim + 2]
        x = big[:, 3:dim + 3]
        keep = check(sporder.dropout(x, 0.4, 8, offset=1), x, 0.4, 8, 1)
        check(sporder.dropout(x, 0.4, 8, offset=1, residual=res), x, 0.4, 8, 1, res)
        t = x.t().contiguous().t()
        assert torch.equal(check(sporder.dropout(t, 0.4, 8, offset=1), t, 0.4, 8, 1), keep)
        flat = torch.randn(rows * dim + 1, device="cuda", generator=g).to(dtype)[1:].view(rows, dim)
        assert torch.equal(check(sporder.dropout(flat, 0.4, 8, offset=1), flat, 0.4, 8, 1), keep)
        row = x[:1].expand(rows, dim)
        check(sporder.dropout(row, 0.4, 8, offset=1), row, 0.4, 8, 1)


def test_in_place_and_out(sporder):
    x = torch.randn(1000, 70, device="cuda")
    want = sporder.dropout(x, 0.2, 1)
    out = torch.empty_like(x)
    assert sporder.dropout(x, 0.2, 1, out=out) is out and torch.equal(out, want)
    y, r = x.clone(), torch.randn_like(x)
    both = sporder.dropout(x, 0.2, 1, residual=r)
    assert torch.equal(sporder.dropout(y, 0.2, 1, out=y), want)
    assert torch.equal(sporder.dropout(x, 0.2, 1, residual=r, out=r), both)


def test_dropped_values_do_not_matter(sporder):
    x = torch.randn(10_000, device="cuda")
    keep = check(sporder.dropout(x, 0.5, 6), x, 0.5, 6, 0)
    bad = torch.where(keep, x, torch.tensor([float("nan"), float("inf")], device="cuda").repeat(5000))
    assert torch.equal(sporder.dropout(bad, 0.5, 6), sporder.dropout(x, 0.5, 6))


def test_no_elements_and_one(sporder):
    assert sporder.dropout(torch.zeros(0, 4, device="cuda"), 0.5, 1).shape == (0, 4)
    assert sporder.dropout(torch.zeros(4, 0, device="cuda"), 0.5, 1).shape == (4, 0)
    x = torch.full((), 2.0, device="cuda")
    assert float(sporder.dropout(x, 0.5, 1)) in (0.0, 4.0)


def test_far_elements(sporder):
    """Past 2^32 elements the block number keeps its high word."""
    n = 2**32 + 2**20 + 5
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    out = sporder.dropout(x, 0.5, 21, offset=4, out=x)
    for first in (0, 2**32 - 8, 2**32, 2**32 + 2**20):
        want = random_bits(5, 21, 4, first) >= np.uint64(2**31)
        assert ((out[first:first + 5] != 0).cpu().numpy() == want).all()


def test_state_on_the_gpu_and_graph(sporder):
    """A captured call reads seed and offset when it runs: each replay has its own."""
    x = torch.randn(3000, 50, device="cuda")
    state = torch.tensor([12345, 100], device="cuda")
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert torch.equal(sporder.dropout(x, 0.3, state, offset=7),
                           sporder.dropout(x, 0.3, 12345, offset=107))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        first = sporder.dropout(x, 0.3, state)
        second = sporder.dropout(x, 0.3, state, offset=1)
        state[1] += 2
    torch.cuda.synchronize()
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, sporder.dropout(x, 0.3, 12345, offset=100 + 2 * k))
        assert torch.equal(second, sporder.dropout(x, 0.3, 12345, offset=101 + 2 * k))


def test_negative_state_words_wrap(sporder):
    x = torch.randn(999, device="cuda")
    state = torch.tensor([-1, -3], device="cuda")
    assert torch.equal(sporder.dropout(x, 0.3, state, offset=5),
                       sporder.dropout(x, 0.3, 2**64 - 1, offset=2))


def test_autograd(sporder):
    """The gradient is dropped and scaled as the value was; a residual's passes."""
    x = torch.randn(50, 40, device="cuda", requires_grad=True)
    r = torch.randn(50, 40, device="cuda", requires_grad=True)
    up = torch.randn(50, 40, device="cuda")
    y = nn.dropout(x, 0.25, 9, offset=3, residual=r)
    y.backward(up)
    assert torch.equal(y, sporder.dropout(x, 0.25, 9, offset=3, residual=r))
    assert torch.equal(x.grad, sporder.dropout(up, 0.25, 9, offset=3))
    assert torch.equal(r.grad, up)
    state = torch.tensor([9, 1], device="cuda")
    x.grad = None
    y = nn.dropout(x, 0.25, state, offset=2)
    state += 5  # the backward pass keeps what the forward pass read
    y.backward(up)
    assert torch.equal(x.grad, sporder.dropout(up, 0.25, 9, offset=3))
    assert nn.dropout(x, 0.25, 9, training=False) is x
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(
            (nn.dropout(x, 0.5, 1) ** 2).sum(), x, create_graph=True)[0].sum(), x)


def test_module_draws_anew(sporder):
    drop = nn.Dropout(0.5, seed=4).to("cuda")
    x = torch.ones(4000, device="cuda", requires_grad=True)
    a = drop(x)
    b = drop(x)
    assert not torch.equal(a, b)
    b.sum().backward()
    assert torch.equal(x.grad, b)
    assert torch.equal(a, sporder.dropout(x, 0.5, 4, offset=0))
    assert torch.equal(b, sporder.dropout(x, 0.5, 4, offset=1))
    again = nn.Dropout(0.5).to("cuda")
    again.load_state_dict(drop.state_dict())
    assert torch.equal(drop(x), again(x))
    drop.eval()
    assert drop(x) is x


def test_refusals(sporder):
    x = torch.zeros(4, 6, device="cuda")
    for bad, err in [(dict(x=x.cpu()), TypeError), (dict(x=x.double()), TypeError),
                     (dict(p=-0.1), ValueError), (dict(p=1.1), ValueError),
                     (dict(p=float("nan")), ValueError), (dict(seed=-1), ValueError),
                     (dict(seed=2**64), ValueError), (dict(offset=-1), ValueError),
                     (dict(offset=2**63), ValueError), (dict(residual=x[:3]), ValueError),
                     (dict(residual=x.half()), TypeError), (dict(residual=x.cpu()), TypeError),
                     (dict(out=x[:, :3]), ValueError), (dict(out=x.half()), ValueError),
                     (dict(seed=torch.zeros(2, dtype=torch.int64)), ValueError),
                     (dict(seed=torch.zeros(3, dtype=torch.int64, device="cuda")), ValueError),
                     (dict(seed=torch.zeros(2, device="cuda")), ValueError)]:
        args = {"x": x, "p": 0.5, "seed": 1, **bad}
        with pytest.raises(err):
            sporder.dropout(args.pop("x"), args.pop("p"), args.pop("seed"), **args)
