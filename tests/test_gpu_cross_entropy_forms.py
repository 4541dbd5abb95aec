"""The linear cross entropy's forms one by one: rows that count nothing beside weights that are
no numbers."""

import pytest
import torch

from test_gpu_cross_entropy import BF16, F16, F32, inputs

pytestmark = pytest.mark.gpu

# Few rows; one pass with a tile for each wave; with tiles shared by the workgroup (16 and 32
# bits, odd and even lengths); tiles.
FORMS = [(F32, 40, 64, 300), (BF16, 20, 64, 300), (F32, 300, 100, 47), (BF16, 300, 64, 16),
         (F32, 300, 101, 47), (BF16, 300, 101, 47), (F32, 300, 256, 60), (BF16, 300, 40, 192),
         (F16, 300, 320, 10), (F32, 300, 7, 47), (F32, 300, 64, 1000), (BF16, 300, 64, 1000)]


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype, rows, dim, classes", FORMS)
def test_rows_that_count_nothing_beside_weights_that_are_no_numbers(sporder, dtype, rows, dim, classes, bad):
    """Their gradients are 0 whatever weights hold."""
    print(f"[forms] {dtype} {rows} {dim} {classes} {bad}", flush=True)
    x, w, t, b, s = inputs(rows, dim, classes, dtype, F32, 0.4, seed=dim)
    t[0], t[1], t[rows - 1] = -100, classes, -100
    w[classes // 2, dim // 3] = bad
    w[0] = -bad
    loss, lse, _ = sporder.linear_cross_entropy(x, w, t, b)
    off = (t < 0) | (t >= classes)
    assert (loss[t == -100] == 0).all() and (lse[t == -100] == 0).all() and loss[1].isnan()
    for given in (None, loss):
        dx = sporder.linear_cross_entropy_grad(s, x, w, t, lse, b, loss=given)[0]
        assert (dx[off] == 0).all()
