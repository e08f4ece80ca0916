"""The checkpoint format at its ends: step bytes that nothing here writes, and the largest error."""
from __future__ import annotations

import numpy as np
import pytest

from orcaml_amd import _lib
from tests import test_gpu_linear_act as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [4, 16, 40, 300])
@pytest.mark.parametrize("infinite", [False, True])
def test_step_bytes_below_7_read_as_7(ctx, rows, infinite):
    """A checkpoint from elsewhere may hold them.  Every reader takes them alike: the kernel for few rows, the tiles, the
    tiles' second pass for what is not finite, the slopes, and the unpacking."""
    rng = np.random.default_rng(rows)
    cols, n = 70, 40
    codes = rng.integers(-127, 128, (rows, cols))
    bytes_ = rng.integers(0, 10, (rows, -(-cols // 32)))
    value = L.value64(codes, np.maximum(bytes_, 7))
    x8 = L.Packed(ctx, rows, cols, L.write_packed(codes, bytes_))
    dy = (rng.standard_normal((rows, n)) * 2.0 ** 100).astype(np.float32)
    if infinite:
        dy[1, 3] = np.inf
    dw = L.Mat(ctx, shape=(cols, n))
    L.backward(ctx, L.Mat(ctx, dy), L.Mat(ctx, shape=(cols, n)), x8=x8, dw=dw)
    with np.errstate(invalid="ignore"):
        want = value.T @ dy.astype(np.float64)
    fine = np.isfinite(want)
    tol = L.product_tol(np.abs(value).T @ np.abs(np.where(np.isfinite(dy), dy, 0)).astype(np.float64), rows)
    got = dw.get()
    np.testing.assert_array_equal(np.isfinite(got), fine)
    L.close(np.where(fine, got, 0), np.where(fine, want, 0), tol, "dw")
    out = L.Mat(ctx, shape=(rows, cols))
    _lib.call("orca_hip_act8_unpack", ctx.handle, x8.ptr, rows, cols, _lib.F32, out.ptr, cols)
    np.testing.assert_array_equal(out.get(), value.astype(np.float32))


def test_the_largest_error_of_a_checkpoint(ctx):
    """Half a step is the most where the group's largest value is 127.5 of the step below: 1 / 127.5 of that value,
    a little more than 2^-7."""
    step = 2.0 ** -6
    x = np.zeros((1, 32), np.float32)
    x[0, 0], x[0, 1] = 127.5 * step, 0.9999 * step  # too large for that step by half a code: the step doubles
    X, p, out = L.Mat(ctx, x), L.Packed(ctx, 1, 32), L.Mat(ctx, shape=(1, 32))
    _lib.call("orca_hip_act8_pack", ctx.handle, X.ptr, 1, 32, 32, p.ptr)
    _lib.call("orca_hip_act8_unpack", ctx.handle, p.ptr, 1, 32, _lib.F32, out.ptr, 32)
    err = np.abs(out.get() - x.astype(np.float64)).max() / x.max()
    assert 2.0 ** -7 < err <= 1 / 127.5
