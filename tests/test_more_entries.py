"""The C entries of dropout, the norms around a block and the linear cross
entropy without a GPU: what they refuse before anything is queued, the scratch
they ask for, calls with nothing to do and the kernels' registers."""

import ctypes

import pytest

from chunkedgreedy_amd import _lib
from test_kernel_resources import kernels  # noqa: F401 (a fixture)

# An address that no call here may follow: every call is refused, or has
# nothing to do.
P = 1 << 40
F32, BF16, F16 = _lib.TYPE_F32, _lib.TYPE_BF16, _lib.TYPE_F16

DROPOUT = dict(stream=0, type=F32, rows=0, dim=4, x_stride=4, x=P, residual_stride=4, residual=P,
               p=0.5, seed=1, offset=0, state=0, out_stride=4, out=P)
BLOCK = dict(stream=0, type=BF16, vector_type=F32, rows=0, dim=4, x_stride=4, x=P,
             residual_stride=4, residual=P, gate_by_row=1, gate_stride=4, gate=P, post_weight=P,
             weight=P, scale=1.0, eps=1e-5, post_norm=1, y_stride=4, y=P, h_stride=4, h=P,
             post_rstd=P, rstd=P)
BLOCK_GRAD = dict(stream=0, type=BF16, vector_type=F32, rows=0, dim=4, dy_stride=4, dy=P,
                  dh_stride=4, dh=P, x_stride=4, x=P, y_stride=4, y=P, post_rstd=P, rstd=P,
                  gate_by_row=1, gate_stride=4, gate=P, post_weight=0, weight=0, scale=1.0,
                  post_norm=1, dx_stride=4, dx=P, dresidual_stride=4, dresidual=P, dgate_stride=4,
                  dgate=P, dpost_weight=0, dweight=0, work=0, size=0)
LOSS = dict(stream=0, type=F32, rows=2, dim=8, classes=6, x_stride=8, x=P, weight_stride=8,
            weight=P, bias_type=F32, bias=P, target_bits=64, targets=P, ignore=-100, loss=P, lse=P,
            sums=P, work=P, size=1 << 40)
LOSS_GRAD = dict(stream=0, type=F32, rows=2, dim=8, classes=6, grad_stride=1, grad=P, x_stride=8,
                 x=P, weight_stride=8, weight=P, bias_type=F32, bias=P, target_bits=64, targets=P,
                 ignore=-100, lse=P, dx_stride=8, dx=P, dweight_type=F32, dweight_stride=8,
                 dweight=P, dbias=P, work=P, size=1 << 40)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def call(lib, name, args):
    return getattr(lib, name)(*args.values())


@pytest.mark.parametrize("name, good", [("sporder_dropout", DROPOUT),
                                        ("sporder_residual_norm", BLOCK),
                                        ("sporder_residual_norm_grad", BLOCK_GRAD)])
def test_nothing_to_do(lib, name, good):
    """No rows: OK, whatever the pointers.  (The loss of no rows has sums to
    write, and its gradient zeros.)"""
    for kind in (F32, BF16, F16):
        args = {**good, "type": kind}
        assert call(lib, name, args) == _lib.OK
        assert call(lib, name, {k: 0 if v == P else v for k, v in args.items()}) == _lib.OK


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(type=-1), dict(rows=-1), dict(dim=-1), dict(x_stride=-1),
    dict(residual_stride=-1), dict(rows=2, out_stride=3), dict(p=-0.1), dict(p=1.5),
    dict(p=float("nan")), dict(offset=1 << 63), dict(rows=1, x=0), dict(rows=1, out=0)])
def test_dropout_refuses(lib, bad):
    assert call(lib, "sporder_dropout", {**DROPOUT, **bad}) == _lib.BAD_ARGUMENT


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(vector_type=3), dict(rows=-1), dict(dim=0), dict(dim=2**23 + 1),
    dict(x_stride=-1), dict(residual_stride=-1), dict(gate_stride=-1), dict(rows=2, y_stride=3),
    dict(rows=2, h_stride=3), dict(eps=-1.0), dict(eps=float("nan")), dict(post_norm=0),
    dict(rows=1, x=0), dict(rows=1, y=0), dict(rows=1, h=0), dict(rows=1, post_rstd=0),
    dict(rows=1, rstd=0)])
def test_block_refuses(lib, bad):
    """post_norm=0 with a post_weight is refused too."""
    assert call(lib, "sporder_residual_norm", {**BLOCK, **bad}) == _lib.BAD_ARGUMENT


@pytest.mark.parametrize("bad", [
    dict(type=3), dict(vector_type=-1), dict(rows=-1), dict(dim=0), dict(dim=2**23 + 1),
    dict(dy_stride=-1), dict(dh_stride=-1), dict(x_stride=-1), dict(y_stride=-1),
    dict(gate_stride=-1), dict(rows=2, dx_stride=3), dict(rows=2, dresidual_stride=3),
    dict(rows=2, dgate_stride=3), dict(rows=1, x=0), dict(rows=1, y=0), dict(rows=1, rstd=0),
    dict(rows=1, dx=0), dict(rows=1, dresidual=0), dict(rows=1, dgate=0),
    dict(rows=1, weight=P, dweight=P), dict(rows=1, weight=P, dweight=P, work=P, size=15),
    dict(rows=1, weight=P, dweight=P, work=P + 4, size=1 << 20)])
def test_block_grad_refuses(lib, bad):
    assert call(lib, "sporder_residual_norm_grad", {**BLOCK_GRAD, **bad}) == _lib.BAD_ARGUMENT


COMMON = [
    dict(type=3), dict(bias_type=3), dict(target_bits=16), dict(rows=-1), dict(dim=0),
    dict(dim=65537), dict(classes=0), dict(classes=2**25 + 1), dict(x_stride=-1),
    dict(weight_stride=-1), dict(rows=2**37 + 1), dict(rows=2**23 - 255, classes=1000),
    dict(rows=2**23 - 255, dim=7), dict(rows=2**20, classes=2**18), dict(x=0), dict(weight=0),
    dict(targets=0), dict(work=0), dict(work=P + 128), dict(classes=50_000, size=1000)]


@pytest.mark.parametrize("bad", COMMON + [dict(loss=0), dict(lse=0), dict(sums=0)])
def test_loss_refuses(lib, bad):
    assert call(lib, "sporder_linear_cross_entropy", {**LOSS, **bad}) == _lib.BAD_ARGUMENT


@pytest.mark.parametrize("bad", COMMON + [
    dict(dweight_type=BF16), dict(type=BF16, dweight_type=F16), dict(grad_stride=-1),
    dict(dx_stride=7), dict(dweight_stride=7), dict(grad=0), dict(lse=0), dict(dx=0),
    dict(dweight=0)])
def test_loss_grad_refuses(lib, bad):
    assert call(lib, "sporder_linear_cross_entropy_grad", {**LOSS_GRAD, **bad}) == _lib.BAD_ARGUMENT


def test_scratch(lib):
    """No rows and refused sizes need none; the loss's stays below the logits it
    doesn't keep, the packed operands and a few numbers a row."""
    assert lib.sporder_residual_norm_grad_work_bytes(0, 64) == 0
    assert lib.sporder_residual_norm_grad_work_bytes(5, 0) == 0
    assert 0 < lib.sporder_residual_norm_grad_work_bytes(10**9, 16384) <= 2**30
    for name in ("sporder_linear_cross_entropy_work_bytes",
                 "sporder_linear_cross_entropy_grad_work_bytes"):
        entry = getattr(lib, name)
        assert entry(BF16, 0, 64, 10, 64, P, 64, P) == 0
        assert entry(BF16, 10, 0, 10, 64, P, 64, P) == 0
        assert entry(7, 10, 64, 10, 64, P, 64, P) == 0
    forward = lib.sporder_linear_cross_entropy_work_bytes
    # aligned 16-bit operands are read where they lie
    assert forward(BF16, 16384, 2048, 50_000, 2048, P, 2048, P) < 2**27
    # others are packed
    assert forward(BF16, 16384, 2047, 50_000, 2047, P, 2047, P) > 2 * (16384 + 50_000) * 2047
    # few classes need sums by workgroup only
    assert forward(F32, 2_000_000, 128, 47, 128, P, 128, P) < 2**20
    assert lib.sporder_linear_cross_entropy_grad_work_bytes(
        F32, 2_000_000, 128, 47, 128, P, 128, P) < 2**25


def test_signatures_take_these_arguments():
    for name, args in (("sporder_dropout", DROPOUT), ("sporder_residual_norm", BLOCK),
                       ("sporder_residual_norm_grad", BLOCK_GRAD),
                       ("sporder_linear_cross_entropy", LOSS),
                       ("sporder_linear_cross_entropy_grad", LOSS_GRAD)):
        kinds, result = _lib.SIGNATURES[name]
        assert result is ctypes.c_int32 and len(kinds) == len(args)


def test_kernels_spill_no_vector_registers(kernels):  # noqa: F811
    """All but the largest tiles of two 16-bit halves per operand, whose
    accumulators take half of the registers."""
    found = 0
    for name, k in kernels.items():
        if not any(part in name for part in ("dropout", "block_norm", "few_", "narrow_", "ce_")):
            continue
        found += 1
        if "Li2ENS" in name and "ELi4ELi4ELi2E" in name:
            assert k["vgpr_spill_count"] <= 32, name
        else:
            assert k["vgpr_spill_count"] == 0 and k["private_segment_fixed_size"] == 0, name
    assert found > 50
