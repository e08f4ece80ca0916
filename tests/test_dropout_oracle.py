"""The oracle's Philox4x32-10 against the published vectors of its authors' test suite."""
from __future__ import annotations

import numpy as np
import pytest

from tests.norm_oracle import dropout_factor, philox


@pytest.mark.parametrize("counter,key,words", [
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])])
def test_known_words(counter, key, words):
    assert [int(w) for w in philox(counter, key)] == words


def test_the_share_kept():
    """512 x 1024 values: a binomial's deviation is below sqrt(0.25 / 2^19) = 0.0007; five of them."""
    for p in (0.1, 0.5, 0.9):
        kept = (dropout_factor(512, 1024, p, 7, 9) > 0).mean()
        assert abs(kept - (1 - p)) < 0.0035
    assert np.all(dropout_factor(3, 5, 1.0, 1, 2) == 0) and np.all(dropout_factor(3, 5, 2.0 ** -34, 1, 2) == 1)
