"""Sums along very long rows: a chain of n additions of one value to itself is off by up to n U / 2 relative where the value
lies just below half a step of the sum above a multiple of its step, as the squares here do for some length of chain."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from orcaml_amd import _lib
from tests.norm_oracle import U
from tests.test_gpu_norm import params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [2 ** 20 + 3, 2 ** 24 + 2])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_long_rows(ctx, cols, kind):
    """Rows of +c and -c in turn.  A thread has 2^14 quads of a row of 2^24 values: 64 quads a run, 256 runs, so a
    square goes through 4 * 64 + 256 additions and 16 over the threads; r is off by half of that."""
    print(f"long rows {cols} {kind}", flush=True)
    eps, quads = 1e-5, cols / 1024
    chain = 4 * 64 + quads / 64 + 20
    for k in (6, 8, 10):
        c = np.float32(np.sqrt(1 + 0.49 * 2.0 ** -k))
        host = np.full((2, cols), c, np.float32)
        host[:, 1::2] = -c
        if cols % 2:
            host[:, -1] = 0  # the mean is 0
        x, y, dx = ctx.upload(host), ctx.alloc(8 * cols), ctx.alloc(8 * cols)
        p = params(kind, None, None, eps)
        _lib.call("orca_hip_norm", ctx.handle, 2, cols, x.ptr, cols, ctypes.byref(p), y.ptr, cols, None)
        square = np.float64(c) ** 2 * (cols // 2 * 2) / cols
        r = 1 / np.sqrt(square + np.float64(np.float32(eps)))
        got = y.download(count=2 * cols).reshape(2, cols)
        err = float(np.abs(got - host * r).max()) / U
        print("y", err, flush=True)
        assert err <= chain / 2 + 10
        # dy = unit(x): dx = r (unit - unit mean(unit^2)), a difference of nearly equal numbers of about 1, whose
        # second one is off by the chain, once from its own sum and once from r^2
        _lib.call("orca_hip_norm_backward", ctx.handle, 2, cols, y.ptr, cols, x.ptr, cols, ctypes.byref(p), None, 0, dx.ptr,
                  cols, None, None)
        u = host * r
        want = r * (u - u * (square * r * r))
        err = float(np.abs(dx.download(count=2 * cols).reshape(2, cols) - want).max()) / U
        print("dx", err, flush=True)
        assert err <= 3 * chain + 40
