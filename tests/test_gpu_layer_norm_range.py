"""Layer norm's gradients of rows whose mean times rstd is past 32 bits: every
(x - mean) rstd of the row is finite, and so is the result, whatever lies past
the row's end in the lanes that hold it."""

import pytest
import torch

from test_gpu_layer_norm import check_backward, inputs

pytestmark = pytest.mark.gpu


# Constant rows of a power of two: their sums, mean and (zero) variance are
# exact, rstd is eps^-1/2, and 2^120 * 316 and 2^110 * 1e6 pass 2^128.
@pytest.mark.parametrize("dim", [1, 3, 17, 31, 33, 63, 65, 100, 101, 128, 129, 130, 257, 516, 1001,
                                 1028, 2050, 4100, 8200, 16000, 16390])
def test_constant_rows_far_from_zero(sporder, dim):
    for power, eps in ((120, 1e-5), (110, 1e-12)):
        if dim * 2.0**power >= 2.0**127:
            continue
        for dtype, wtype in ((torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                             (torch.bfloat16, torch.bfloat16)):
            x, g, w, b = inputs(5, dim, dtype, wtype, seed=dim)
            x[1], x[3:] = 2.0**power, -(2.0**power)
            got = sporder.layer_norm(x, w, b, eps=eps)
            assert torch.equal(got[1][[1, 3, 4]].double(), x[[1, 3, 4], 0].double())
            for rows in (slice(0, 5), slice(1, 2)):
                grads = sporder.layer_norm_grad(g[rows], x[rows], got[1][rows], got[2][rows], w)
                assert all(t.isfinite().all() for t in grads)
                check_backward(grads, g[rows], x[rows], got[1][rows], got[2][rows], w)
            # Rows that start off every vector.
            apart = torch.empty(2, 5 * (dim + 1) + 1, device="cuda", dtype=dtype)
            xs, gs = (flat[1:].view(5, dim + 1)[:, :dim] for flat in apart)
            xs.copy_(x)
            gs.copy_(g)
            grads = sporder.layer_norm_grad(gs, xs, got[1], got[2], w)
            check_backward(grads, g, x, got[1], got[2], w)
