"""Norms, joints and dropout where 32 bits do not reach: rows more than 2^32 bytes and 2^31 elements apart, operands beyond
the memory-side cache, more rows than a launch has blocks."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from orcaml_amd import _lib
from tests import norm_oracle as O
from tests.test_gpu_norm import Joint, Matrix, close, params

pytestmark = pytest.mark.gpu


@pytest.fixture
def room(ctx):
    """Device memory of earlier tests given back first, this one's afterwards."""
    ctx.sync()
    ctx.empty_cache()
    yield ctx
    ctx.sync()
    ctx.empty_cache()


class Far:
    """A matrix of few rows whose rows are `ld` apart; only what stands near the rows is written and read."""

    PAD = 8

    def __init__(self, ctx, rows, cols, ld, values=None):
        self.ctx, self.rows, self.cols, self.ld = ctx, rows, cols, ld
        self.buf = ctx.alloc(4 * ((rows - 1) * ld + cols + 2 * self.PAD))
        self.ptr = self.buf.ptr + 4 * self.PAD
        for r in range(rows):
            line = np.full(cols + 2 * self.PAD, Matrix.GAP, np.float32)
            if values is not None:
                line[self.PAD:-self.PAD] = values[r]
            self._copy("orca_hip_h2d", r, line)

    def _copy(self, call, r, line):
        at, host = self.buf.ptr + 4 * r * self.ld, line.ctypes.data_as(ctypes.c_void_p)
        _lib.call(call, self.ctx.handle, *((at, host) if call == "orca_hip_h2d" else (host, at)), line.nbytes)

    def read(self):
        out = np.empty((self.rows, self.cols + 2 * self.PAD), np.float32)
        for r in range(self.rows):
            self._copy("orca_hip_d2h", r, out[r])
        assert (out[:, :self.PAD] == Matrix.GAP).all() and (out[:, -self.PAD:] == Matrix.GAP).all()
        return out[:, self.PAD:-self.PAD].copy()


class FarJoint(Joint):
    LD = 2 ** 31 + 9

    def matrix(self, values=None, rows=None):
        rows = values.shape[0] if values is not None else rows if rows is not None else self.m
        return Far(self.ctx, rows, self.n, self.LD, values)

    def backward(self, y, **kw):
        self.pad = self.LD - self.n  # the results' leading dimension
        return super().backward(y, **kw)


# rows in passes, of one wave, of four and eight; one gate row for each row, so that it has far rows as well
@pytest.mark.parametrize("n", [3, 260, 1501, 5000, 9001])
def test_rows_far_apart(room, n):
    print(f"far rows {n}", flush=True)
    j = FarJoint(room, n, 2, n, "layer", "rms", 2, 0.2)
    j.check()
    rng = np.random.default_rng(n)
    x = rng.standard_normal((2, n)).astype(np.float32)
    del j
    mx, my = Far(room, 2, n, FarJoint.LD, x), Far(room, 2, n, FarJoint.LD)
    _lib.call("orca_hip_dropout", room.handle, 2, n, mx.ptr, mx.ld, 0.5, 7, 3, my.ptr, my.ld)
    np.testing.assert_array_equal(my.read(), x * O.dropout_factor(2, n, 0.5, 7, 3).astype(np.float32))
    p = params("layer", None, None)
    _lib.call("orca_hip_norm", room.handle, 2, n, mx.ptr, mx.ld, ctypes.byref(p), my.ptr, my.ld, None)
    x64 = x.astype(np.float64)
    y = my.read()
    close(y, O.norm("layer", x64, 1e-5, np.ones(n), np.zeros(n)), "y")
    _lib.call("orca_hip_norm_backward", room.handle, 2, n, my.ptr, my.ld, mx.ptr, mx.ld, ctypes.byref(p), None, 0,
              (dx := Far(room, 2, n, FarJoint.LD)).ptr, dx.ld, None, None)
    close(dx.read(), O.norm_back("layer", x64, 1e-5, np.ones(n), y.astype(np.float64))[0], "dx")


def kept(rows, cols, seed, offset, border=2 ** 31):
    """Which values of the given rows a dropout with p = 1/2 keeps."""
    rows, quads = np.asarray(rows, np.uint64), -(-cols // 4)
    q = np.broadcast_to(np.arange(quads, dtype=np.uint64)[None], (rows.size, quads))
    r = np.broadcast_to(rows[:, None], q.shape)
    zero = np.zeros(q.shape, np.uint64)
    w = O.philox([q, r, zero + np.uint64(offset), zero], [seed, 0])
    return np.stack(w, 2).reshape(rows.size, 4 * quads)[:, :cols] >= border


# just below 256 MiB of operands and from there on, where the loads are others
@pytest.mark.parametrize("m,n", [(8184, 4099), (8200, 4099), (8195, 4096), (11200000, 3), (5600000, 6)])
@pytest.mark.parametrize("pad,start", [(0, 0), (3, 1)])
def test_dropout_beyond_the_cache(room, m, n, pad, start):
    print(f"dropout {m} x {n} pad {pad}", flush=True)
    rng = np.random.default_rng(m)
    x = rng.standard_normal((m, n), dtype=np.float32)
    mx, my = Matrix(room, m, n, x, n + pad, start), Matrix(room, m, n, None, n + pad, start)
    _lib.call("orca_hip_dropout", room.handle, m, n, mx.ptr, mx.ld, 0.5, 11, 5, my.ptr, my.ld)
    got = my.read()
    assert ((got == 0) | (got == 2 * x)).all()
    rows = np.unique(np.concatenate([np.arange(40), m - 1 - np.arange(40), rng.integers(0, m, 400)]))
    np.testing.assert_array_equal(got[rows], 2 * x[rows] * kept(rows, n, 11, 5))
    _lib.call("orca_hip_dropout", room.handle, m, n, mx.ptr, mx.ld, 0.5, 11, 5, mx.ptr, mx.ld)
    np.testing.assert_array_equal(mx.read(), got)


def test_dropout_of_more_rows_than_blocks(room):
    """A launch has 2^23 blocks of rows at most, here of one row each; 2^32 elements in place."""
    m, n = 2 ** 23 + 5, 513
    buf = room.alloc(4 * m * n)
    room.fill(buf, 1.0, m * n)
    _lib.call("orca_hip_dropout", room.handle, m, n, buf.ptr, n, 0.5, 77, 5, buf.ptr, n)
    for r in (0, 1, 2 ** 22, 2 ** 23 - 1, 2 ** 23, m - 1):
        line = np.empty(n, np.float32)
        _lib.call("orca_hip_d2h", room.handle, line.ctypes.data_as(ctypes.c_void_p), buf.ptr + 4 * r * n, line.nbytes)
        np.testing.assert_array_equal(line, 2.0 * kept([r], n, 77, 5)[0])
