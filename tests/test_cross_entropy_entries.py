"""The linear cross entropy's C entries without a GPU: the entry that takes the losses
refuses what the one without them refuses."""

import ctypes

import pytest

from chunkedgreedy_amd import _lib
from test_more_entries import COMMON, LOSS, LOSS_GRAD, P, call, lib  # noqa: F401 (a fixture)

BF16, F16 = _lib.TYPE_BF16, _lib.TYPE_F16
OF_LOSS = {}
for name, value in LOSS_GRAD.items():
    OF_LOSS[name] = value
    if name == "lse":
        OF_LOSS["loss"] = P


@pytest.mark.parametrize("bad", COMMON + [
    dict(dweight_type=BF16), dict(type=BF16, dweight_type=F16), dict(grad_stride=-1),
    dict(dx_stride=7), dict(dweight_stride=7), dict(grad=0), dict(lse=0), dict(dx=0),
    dict(dweight=0)])
def test_gradient_of_losses_refuses(lib, bad):  # noqa: F811
    name = "sporder_linear_cross_entropy_grad_of_loss"
    kinds, result = _lib.SIGNATURES[name]
    assert result is ctypes.c_int32 and len(kinds) == len(OF_LOSS)
    for loss in (P, 0):
        assert call(lib, name, {**OF_LOSS, "loss": loss, **bad}) == _lib.BAD_ARGUMENT


GB = 2**30
F32 = _lib.TYPE_F32


@pytest.mark.parametrize("kind, rows, dim, classes", [
    (F32, 2_449_029, 128, 193), (F32, 2_449_029, 128, 1000), (F32, 2_449_029, 256, 172),
    (F32, 580_000, 500, 172), (BF16, 580_000, 500, 172), (F32, 8_000_000, 100, 300),
    (BF16, 8_000_000, 64, 1000), (BF16, 8_000_000, 65, 1000), (F32, 2**23 - 256, 16, 2**14),
    (BF16, 2**23 - 256, 8, 2**14), (BF16, 300_000, 4096, 50_000), (F32, 300_000, 4096, 50_000),
    (F16, 16_384, 4096, 60_000), (BF16, 256, 4096, 131_072), (F32, 100, 65_536, 100_000),
    (BF16, 2000, 65_536, 200_000), (F32, 131_072, 300, 1000), (F32, 131_073, 300, 1000)])
def test_scratch_of_the_gradients_is_bounded(lib, kind, rows, dim, classes):  # noqa: F811
    """Rows and classes are cut into pieces of which g in either order, the packed rows, both
    turned operands and dx's sums take at most half a GB each (dx's one), and column maxima
    another half; beside them w packed, dw's sums over the pieces of the rows and some numbers a
    row and class."""
    entry = lib.sporder_linear_cross_entropy_grad_work_bytes
    for at in (P, P + 2):  # 16-bit operands read where they lie, and packed
        size = entry(kind, rows, dim, classes, dim, at, dim, at)
        whole = (dim + 63) // 64 * 64
        limit = 4 * GB + classes * (2 * 4 * whole + 8) + 40 * rows
        assert 0 < size <= limit, (size / GB, limit / GB)
        if rows >= 131_072 and classes <= 1000:  # below 2.1 GB however many rows
            assert size <= 2.1 * GB + 40 * rows, size / GB


SHAPES = [(classes, dim) for classes in (1, 16, 17, 32, 47, 48, 49, 64, 65, 90, 96, 97, 128, 129, 172, 192, 193, 1000)
          for dim in (7, 8, 64, 100, 128, 129, 192, 193, 256, 257, 384, 385, 512, 513)]


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_both_directions_take_the_same_rows(lib, kind):  # noqa: F811
    """Every number of rows that the forward call takes its gradients take, and the
    Python check tells which."""
    import torch

    from chunkedgreedy_amd.sporder import _train

    dtype = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}[kind]
    for classes, dim in SHAPES:
        for rows in (2**23 - 256, 2**23 - 255, 10_000_000, 2**31 - 1024, 2**37 // classes, 2**37 // classes + 1):
            taken = [entry(kind, rows, dim, classes, dim, P, dim, P) > 0 for entry in (
                lib.sporder_linear_cross_entropy_work_bytes,
                lib.sporder_linear_cross_entropy_grad_work_bytes)]
            assert taken[0] == taken[1], (classes, dim, rows)
            small = rows <= 2**23 - 256 and rows * classes <= 2**37
            if rows <= 2**31 - 1024:
                assert taken[0] == (small or _train._one_pass(dtype, dim, classes)), (classes, dim, rows)
            for name, good in (("sporder_linear_cross_entropy", LOSS), ("sporder_linear_cross_entropy_grad", LOSS_GRAD)):
                if not taken[0]:
                    bad = dict(type=kind, rows=rows, dim=dim, classes=classes, x_stride=dim, weight_stride=dim)
                    more = {"dweight_type": kind, "dx_stride": dim, "dweight_stride": dim} if "dx" in good else {}
                    assert call(lib, name, {**good, **bad, **more}) == _lib.BAD_ARGUMENT
