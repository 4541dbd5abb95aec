"""The seeds that nn.Dropout takes, without a GPU."""

import pytest

from chunkedgreedy_amd import nn


@pytest.mark.parametrize("seed", [0, 5, 2**63 - 1, 2**63, 2**64 - 1, -1])
def test_seeds_are_kept_as_64_bits(seed):
    """All that sporder.dropout takes; a negative one is its 64 bits."""
    state = nn.Dropout(0.5, seed).state.tolist()
    assert state[0] % 2**64 == seed % 2**64 and state[1] == 0


@pytest.mark.parametrize("seed", [2**64, -(2**63) - 1])
def test_other_seeds_are_refused(seed):
    with pytest.raises(ValueError):
        nn.Dropout(0.5, seed)
