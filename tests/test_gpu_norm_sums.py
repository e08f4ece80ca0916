"""Sums over very many rows.

A chain of n additions of one value v to itself is off by up to n U / 2 relative, if v lies just below half a step of the sum
above a multiple of its step: each addition then drops nearly half a step.  The values here are such for chains of
many lengths (1 + 0.49 2^-k; one k a column), and no bound below grows with the number of rows."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from orcaml_amd import _lib
from tests.norm_oracle import U
from tests.test_gpu_norm import params

pytestmark = pytest.mark.gpu


def worst(cols, low=4):
    """Values for chains of 2^low additions and on."""
    return (1 + 0.49 * 2.0 ** -(low + np.arange(cols) % 12)).astype(np.float32)


def rows_of(ctx, rows, v):
    return ctx.upload(np.broadcast_to(v, (rows, v.size)))


# Additions that a term goes through: 512 rows in a chain, or twice that where whole groups of rows are; then those of
# the partial sums: of 32768, 64 eights in a thread's chain, and 3 + 3 + 8 over eights, a wave and the waves.
BOUND = 2 * 512 + 64 + 14 + 10


@pytest.mark.parametrize("rows,cols,low", [(2 ** 24 + 3, 3, 8), (2 ** 23 + 1, 1, 10),
                                                (2 ** 25 + 5, 4, 10), (2 ** 25, 4, 13)])
def test_bias_and_weight(ctx, rows, cols, low):
    print(f"sums {rows} x {cols}", flush=True)
    v = worst(cols, low)
    dy, x, p = rows_of(ctx, rows, v), ctx.alloc(4 * rows * cols), params("rms", None, None)
    ctx.fill(x, 2.0, rows * cols)
    dw, db = ctx.alloc(4 * cols), ctx.alloc(4 * cols)
    _lib.call("orca_hip_norm_backward", ctx.handle, rows, cols, dy.ptr, cols, x.ptr, cols, ctypes.byref(p), None, 0, None,
              0, dw.ptr, db.ptr)
    want = rows * v.astype(np.float64)
    err = np.abs(db.download(count=cols) / want - 1) / U
    print("db", err.max(), flush=True)
    assert (err <= BOUND).all(), err
    unit = 2 / np.sqrt(4 + np.float64(np.float32(1e-5)))
    err = np.abs(dw.download(count=cols) / (want * unit) - 1) / U
    print("dw", err.max(), flush=True)
    assert (err <= BOUND + 10).all(), err  # unit is off by less than ten roundings


@pytest.mark.parametrize("rows,cols,groups,low", [
    (2 ** 23, 3, 1, 8), (2 ** 23, 3, 4, 8), (2 ** 23, 2, 512, 9),
    (2 ** 25, 4, 1, 11), (2 ** 25, 4, 1024, 11), (2 ** 24, 4, 1 << 20, 2)])
def test_gate(ctx, rows, cols, groups, low):
    """A gate for all rows, some groups, and more groups than blocks, of many rows each."""
    print(f"gate sums {rows} x {cols} groups {groups}", flush=True)
    v = worst(cols, low)
    dy, f, gate = rows_of(ctx, rows, v), ctx.alloc(4 * rows * cols), rows_of(ctx, groups, v)
    ctx.fill(f, 2.0, rows * cols)
    dgate = ctx.alloc(4 * groups * cols)
    b = _lib.ResidualBlock(gate=gate.ptr, groups=groups, ldgate=cols, residual_scale=1.0, block_scale=1.0)
    g = _lib.ResidualGrads(dgate=dgate.ptr, lddgate=cols)
    _lib.call("orca_hip_residual_norm_backward", ctx.handle, rows, cols, dy.ptr, cols, None, cols, f.ptr, cols, None, cols,
              ctypes.byref(b), ctypes.byref(g))
    want = rows // groups * 2 * v.astype(np.float64)
    err = np.abs(dgate.download(count=groups * cols).reshape(groups, cols) / want - 1) / U
    print("dgate", err.max(), flush=True)
    assert (err <= BOUND).all(), err.max()


@pytest.mark.parametrize("rows,cols,groups", [(2 ** 18 + 600, 1028, 0), (2 ** 18, 1028, 1024)])
def test_more_rows_than_a_block_adds_up(ctx, rows, cols, groups):
    """Four waves a row: every gradient of all the blocks' rows, by rows that repeat."""
    print(f"many blocks {rows} x {cols}", flush=True)
    n = rows * cols
    dy, f, du, y = (ctx.alloc(4 * n) for _ in range(4))
    v = 1 + 0.49 * 2.0 ** -9
    for buf, value in ((dy, v), (f, 2.0), (du, 0.5), (y, 4.0)):
        ctx.fill(buf, value, n)
    names = ("dpost_weight", "dpost_bias", "dnext_weight", "dnext_bias")
    out = {k: ctx.alloc(4 * cols) for k in names}
    gate = rows_of(ctx, groups, np.ones(cols, np.float32)) if groups else None
    if groups:
        out["dgate"] = ctx.alloc(4 * groups * cols)
    eps = 1.0
    b = _lib.ResidualBlock(post=params("rms", None, None, eps), next=params("rms", None, None, eps),
                           gate=gate.ptr if gate else None, groups=groups, ldgate=cols, residual_scale=1.0, block_scale=1.0)
    g = _lib.ResidualGrads(**{k: o.ptr for k, o in out.items()}, lddgate=cols)
    _lib.call("orca_hip_residual_norm_backward", ctx.handle, rows, cols, dy.ptr, cols, du.ptr, cols, f.ptr, cols, y.ptr, cols,
              ctypes.byref(b), ctypes.byref(g))
    uy, uf = 4 / np.sqrt(17), 2 / np.sqrt(5)
    dyt = np.float64(np.float32(v)) + (0.5 - uy * 0.5 * uy) / np.sqrt(17)
    want = {"dnext_bias": rows * 0.5, "dnext_weight": rows * 0.5 * uy, "dpost_bias": rows * dyt, "dpost_weight": rows * dyt * uf,
            "dgate": rows // max(groups, 1) * dyt * uf}
    for k, o in out.items():
        err = np.abs(o.download(count=cols * (groups if k == "dgate" else 1)) / want[k] - 1) / U
        print(k, err.max(), flush=True)
        # a row's sums run over 40 additions at most, and some ten roundings follow
        assert (err <= BOUND + 60).all(), k
