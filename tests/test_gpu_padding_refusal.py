"""A padding row outside the table is refused by the lookup itself, not by a
backward pass after it."""

import pytest
import torch

from chunkedgreedy_amd import nn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("padding", [-1, 10, 2**40])
def test_differentiable_lookup_refuses_padding_outside_the_table(sporder, padding):
    table = torch.randn(10, 4, device="cuda", requires_grad=True)
    tokens = torch.tensor([1, 2], device="cuda")
    with pytest.raises(ValueError):
        nn.embedding(table, tokens, padding_idx=padding)
    with torch.no_grad(), pytest.raises(ValueError):
        nn.embedding(table, tokens, padding_idx=padding)
    with pytest.raises(ValueError):
        sporder.embedding_grad(torch.ones(2, 4, device="cuda"), tokens, 10, padding_idx=padding)
    for row in (0, 9, None):
        nn.embedding(table, tokens, padding_idx=row).sum().backward()
