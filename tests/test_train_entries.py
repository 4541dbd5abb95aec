"""The C entries of the training operators without a GPU: what they refuse
before anything is queued, the scratch they ask for, calls with nothing to do,
the bound on Newton-Schulz coefficients and the kernels' registers."""

import ctypes
import itertools

import numpy as np
import pytest

from chunkedgreedy_amd import _lib
from test_kernel_resources import kernels  # noqa: F401 (a fixture)

# An address that no call here may follow: every call is refused, or has
# nothing to do.
P = 1 << 40
F32, BF16, F16 = _lib.TYPE_F32, _lib.TYPE_BF16, _lib.TYPE_F16


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


LOOKUP = dict(stream=0, type=F32, rows=10, dim=4, table_stride=4, table=P, count=0, bits=32,
              tokens=P, scale=1.0, out_stride=4, out=P)
LOOKUP_GRAD = dict(stream=0, type=F32, count=2, dim=4, grad_stride=4, grad=P, bits=32, tokens=P,
                   scale=1.0, padding=-1, rows=10, out_type=F32, out_stride=4, out=P, work=P,
                   size=1 << 40)
NORM = dict(stream=0, type=F32, weight_type=F32, rows=0, dim=4, x_stride=4, x=P, weight=0, bias=0,
            eps=1e-5, y_stride=4, y=P, mean=P, rstd=P)
NORM_GRAD = dict(stream=0, type=F32, weight_type=F32, rows=0, dim=4, dy_stride=4, dy=P, x_stride=4,
                 x=P, mean=P, rstd=P, weight=0, dx_stride=4, dx=P, dweight=0, dbias=0, work=0,
                 size=0)
ORTHO = dict(stream=0, type=F32, batch=0, rows=8, cols=8, batch_stride=64, stride=8, g=P, steps=5,
             a=3.4445, b=-4.7750, c=2.0315, eps=1e-7, out=P, work=P, size=1 << 40)


@pytest.mark.parametrize("name, good", [("sporder_embedding", LOOKUP),
                                        ("sporder_layer_norm", NORM),
                                        ("sporder_layer_norm_grad", NORM_GRAD),
                                        ("sporder_newton_schulz", ORTHO)])
def test_nothing_to_do(lib, name, good):
    """No tokens, rows or matrices: OK, whatever the pointers."""
    for kind in (F32, BF16, F16):
        args = {**good, "type": kind}
        assert getattr(lib, name)(*args.values()) == _lib.OK
        none = {k: 0 if v in (P, 1 << 40) else v for k, v in args.items()}
        assert getattr(lib, name)(*none.values()) == _lib.OK


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(type=-1), dict(rows=0), dict(dim=0), dict(dim=2**23 + 1), dict(count=-1),
    dict(bits=16), dict(table_stride=-1), dict(count=2, out_stride=3), dict(count=2, table=0),
    dict(count=2, tokens=0), dict(count=2, out=0)])
def test_lookup_refuses(lib, bad):
    assert lib.sporder_embedding(*{**LOOKUP, **bad}.values()) == _lib.BAD_ARGUMENT


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(out_type=BF16), dict(type=BF16, out_type=F16), dict(rows=0),
    dict(rows=2**31 - 1), dict(dim=0), dict(dim=2**23 + 1), dict(count=-1), dict(count=2**28),
    dict(bits=8), dict(grad_stride=-1), dict(out_stride=3), dict(grad=0), dict(tokens=0),
    dict(out=0), dict(count=0, out=0), dict(count=100_000, work=0),
    dict(count=100_000, work=P + 128), dict(count=100_000, size=1 << 10)])
def test_lookup_grad_refuses(lib, bad):
    assert lib.sporder_embedding_grad(*{**LOOKUP_GRAD, **bad}.values()) == _lib.BAD_ARGUMENT


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(weight_type=3), dict(rows=-1), dict(dim=0), dict(dim=2**23 + 1),
    dict(x_stride=-1), dict(rows=2, y_stride=3), dict(eps=-1.0), dict(eps=float("nan")),
    dict(rows=1, x=0), dict(rows=1, y=0), dict(rows=1, mean=0), dict(rows=1, rstd=0)])
def test_norm_refuses(lib, bad):
    assert lib.sporder_layer_norm(*{**NORM, **bad}.values()) == _lib.BAD_ARGUMENT


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(weight_type=-1), dict(rows=-1), dict(dim=0), dict(dim=2**23 + 1),
    dict(x_stride=-1), dict(dy_stride=-1), dict(rows=2, dx_stride=3), dict(rows=1, x=0),
    dict(rows=1, dy=0), dict(rows=1, dx=0), dict(rows=1, mean=0), dict(rows=1, rstd=0),
    dict(rows=1, dweight=P), dict(rows=1, dbias=P, work=P, size=31),
    dict(rows=1, dbias=P, work=P + 4, size=1 << 20)])
def test_norm_grad_refuses(lib, bad):
    assert lib.sporder_layer_norm_grad(*{**NORM_GRAD, **bad}.values()) == _lib.BAD_ARGUMENT


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(batch=-1), dict(batch=2**15 + 1), dict(rows=0), dict(cols=0),
    dict(rows=2**16 + 1), dict(cols=2**16 + 1), dict(stride=-1), dict(batch_stride=-1),
    dict(steps=0), dict(eps=-1.0), dict(eps=float("nan")), dict(a=float("inf")),
    dict(c=float("nan")), dict(batch=1, g=0), dict(batch=1, out=0),
    dict(batch=1, rows=500, cols=500, work=0), dict(batch=1, rows=500, cols=500, work=P + 16),
    dict(batch=1, rows=500, cols=500, size=1000)])
def test_newton_schulz_refuses(lib, bad):
    assert lib.sporder_newton_schulz(*{**ORTHO, **bad}.values()) == _lib.BAD_ARGUMENT


def test_scratch(lib):
    """Few tokens and small matrices need none; more of anything never needs
    less than its own entries take."""
    assert lib.sporder_embedding_grad_work_bytes(0, 10, 4) == 0
    assert lib.sporder_embedding_grad_work_bytes(1000, 1000, 64) == 0
    assert lib.sporder_embedding_grad_work_bytes(1000, 0, 64) == 0
    for count in (10_000, 1_000_000, 100_000_000):
        size = lib.sporder_embedding_grad_work_bytes(count, 1000, 64)
        assert 12 * count <= size <= 80 * count
    assert lib.sporder_layer_norm_grad_work_bytes(0, 4) == 0
    assert lib.sporder_layer_norm_grad_work_bytes(1, 4) == 32
    assert lib.sporder_layer_norm_grad_work_bytes(10**9, 2**23) <= 2**36
    assert lib.sporder_newton_schulz_work_bytes(1, 32, 64) == 0
    assert lib.sporder_newton_schulz_work_bytes(1, 0, 64) == 0
    for rows, cols in ((500, 700), (4096, 4096), (65536, 64), (1, 65536)):
        size = lib.sporder_newton_schulz_work_bytes(1, rows, cols)
        assert size >= 4 * 2 * rows * cols
        assert size == lib.sporder_newton_schulz_work_bytes(1, cols, rows)
        assert lib.sporder_newton_schulz_work_bytes(7, rows, cols) >= 7 * (size - 4096)


def test_coefficient_bound_follows_the_polynomial(lib):
    """Allowed where the maxima over a fine grid of singular values in [0, 1]
    (and of what each step makes of them) stay clear of 31, refused where they
    pass it.  The grid's maximum is within 1 % of the true one, so values
    between 30 and 32 may go either way."""
    values = [-20.0, -4.775, -1.5, 0.0, 0.5, 2.0315, 3.4445, 12.0]
    seen = {True: 0, False: 0}
    for (a, b, c), steps in itertools.product(itertools.product(values, repeat=3), (1, 2, 5)):
        most, top = 0.0, 1.0
        for _ in range(steps):
            s = np.linspace(0.0, top, 4001)
            t = s * s
            new = float(np.abs(a * s + b * s * t + c * s * t * t).max())
            most = max(most, top * top, float(np.abs(b * t + c * t * t).max()), new)
            if most > 1e6:
                break
            top = new
        if 30.0 < most < 32.0:
            continue
        args = {**ORTHO, "steps": steps, "a": a, "b": b, "c": c}
        got = lib.sporder_newton_schulz(*args.values()) == _lib.OK
        assert got == (most <= 31.0), (a, b, c, steps, most)
        seen[got] += 1
    assert min(seen.values()) > 100


def test_signatures_take_these_arguments():
    for name, args in (("sporder_embedding", LOOKUP), ("sporder_embedding_grad", LOOKUP_GRAD),
                       ("sporder_layer_norm", NORM), ("sporder_layer_norm_grad", NORM_GRAD),
                       ("sporder_newton_schulz", ORTHO)):
        kinds, result = _lib.SIGNATURES[name]
        assert result is ctypes.c_int32 and len(kinds) == len(args)


def test_kernels_spill_no_vector_registers(kernels):  # noqa: F811
    found = 0
    for name, k in kernels.items():
        if any(part in name for part in ("embedding", "norm_", "ortho_")):
            found += 1
            assert k["vgpr_spill_count"] == 0 and k["private_segment_fixed_size"] == 0, name
    assert found > 50
