"""GELU and its slope where they are small: relative to the value, not to 1 + |z|."""
from __future__ import annotations

import math

import numpy as np
import pytest
from scipy.special import erfc

from tests import test_gpu_linear_act as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 700])
def test_gelu_keeps_its_tail(ctx, rows):
    """z comes from a product with 1, exact.  GELU is z R(z) exp(-z^2 / 2) with a smooth R.  The exponent is rounded twice
    and its factor once, to a half step each: 2.5 * 2^-24 of z^2 / 2, an absolute error of the exponent and so a
    relative one of the value.  R is nine multiply-adds over a rounded reciprocal, then come the hardware's exponential
    (an ulp) and three products: 16 * 2^-24.  (z itself, rounded to fp32, moves GELU by z^2 * 2^-24 too.)"""
    z = -np.linspace(0.5, 12.5, rows * 40, dtype=np.float64).astype(np.float32).reshape(rows, 40)
    z64 = z.astype(np.float64)
    one = np.ones((1, 1), np.float32)
    cdf = 0.5 * erfc(-z64 / math.sqrt(2))
    pdf = np.exp(-z64 * z64 / 2) / math.sqrt(2 * math.pi)
    tol = L.U * (1.25 * z64 * z64 + 16)
    col = lambda v: L.Mat(ctx, np.ascontiguousarray(v.reshape(-1, 1)))  # noqa: E731
    y = L.forward(ctx, col(z), L.Mat(ctx, one), "gelu").get().reshape(z.shape)
    L.close(y, z64 * cdf, tol * np.abs(z64) * cdf, "gelu")
    for shape in (z.shape, (z.size, 1)):
        dx = L.Mat(ctx, shape=(shape[0], shape[1]))
        eye = np.eye(shape[1], dtype=np.float32)
        L.backward(ctx, L.Mat(ctx, np.ones(shape, np.float32)), L.Mat(ctx, eye), "gelu", z=L.Mat(ctx, z.reshape(shape)), dx=dx)
        # the slope is a difference of the two: relative to their sizes
        L.close(dx.get(), (cdf + z64 * pdf).reshape(shape), ((tol + 4 * L.U) * (cdf - z64 * pdf)).reshape(shape), "slope")
