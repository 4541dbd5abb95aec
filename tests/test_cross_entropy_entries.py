"""The linear cross entropy's C entries without a GPU: the entry that takes the losses
refuses what the one without them refuses."""

import ctypes

import pytest

from chunkedgreedy_amd import _lib
from test_more_entries import COMMON, LOSS_GRAD, P, call, lib  # noqa: F401 (a fixture)

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
