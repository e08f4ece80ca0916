"""A joint of no rows on the tape, over a joint in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from tests import residual_empty as E
from tests.test_residual_scale import Joints


class Gates(Joints):
    """With gates, of which no rows read anything."""

    def residual_norm_backward(self, dy, du, f, y, m, n, b, want=()):
        assert m == 0 and ("dgate" not in want or (b.gate is not None and b.gate.size == b.groups * n))
        sizes = {"dx": 0, "df": 0, "dgate": b.groups * n}
        return {k: np.zeros(sizes.get(k, n), np.float32) for k in want}


@pytest.mark.parametrize("lead,gate", E.SHAPES)
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_no_rows(lead, gate, scale):
    E.check(Gates(), lead, gate, scale)
