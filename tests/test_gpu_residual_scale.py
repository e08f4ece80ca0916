"""A joint's gradients at any residual scale, by its kernels."""
from __future__ import annotations

import pytest

from tests import residual_scale as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", S.SCALES)
@pytest.mark.parametrize("size", S.SIZES)
@pytest.mark.parametrize("read", S.READ)
def test_gradients_at_a_scale(hb, scale, size, read):
    S.check(hb, scale, size, read)
    S.check(hb, scale, size, read, x_grad=False)
