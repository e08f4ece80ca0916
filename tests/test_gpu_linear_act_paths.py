"""The fused Linear's kernels one by one: each tile and K split (fixed through the context's switches),
the kernels for a few rows, the small backward, matrices past 4 GiB, and columns of one matrix."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from orcaml_amd import _lib
from orcaml_amd.device import Context
from tests import test_gpu_linear_act as L

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[(64, 1), (64, 3), (128, 1), (128, 2), (256, 1), (256, 4)],
                ids=lambda p: f"tile{p[0]}-splits{p[1]}")
def tiled(request):
    with pytest.MonkeyPatch.context() as mp:
        mp.setenv("ORCA_HIP_LINEAR_TILE", str(request.param[0]))
        mp.setenv("ORCA_HIP_LINEAR_SPLITS", str(request.param[1]))
        c = Context(0)
    yield c, request.param[0]
    c.close()


# below a tile, across its edges, k below a stage, at whole stages and past them, several splits' worth
TILE_SHAPES = [(1, 1, 1), (5, 3, 2), (33, 70, 16), (64, 64, 64), (130, 100, 129), (260, 300, 70), (300, 257, 400),
               (20, 600, 1030), (520, 40, 257)]


@pytest.mark.parametrize("m,n,k", TILE_SHAPES)
def test_forward_on_each_tile(tiled, m, n, k):
    L.test_forward(tiled[0], m, n, k)


@pytest.mark.parametrize("m,n,k", TILE_SHAPES)
def test_backward_on_each_tile(tiled, m, n, k):
    L.test_backward(tiled[0], m, n, k)


def test_other_inputs_on_each_tile(tiled):
    c = tiled[0]
    L.test_integers_are_exact(c)
    L.test_split_products_are_exact_where_fp32_is(c)
    L.test_in_place_residual_and_gradient(c)
    L.test_leading_dimensions_and_alignment(c)
    L.test_pack_of_infinities_and_nan(c)
    L.test_results_repeat_bit_for_bit(c)
    for m, n, k in ((4, 40, 48), (150, 140, 100), (70, 70, 3000)):
        L.test_infinities_and_nan_come_out_as_from_fp32(c, m, n, k)
    for m, n, k in ((0, 5, 7), (5, 0, 7), (5, 7, 0), (70, 40, 0)):
        L.test_empty_sizes(c, m, n, k)


def names(ctx, run):
    ctx.prof_reset()
    ctx.prof_enable(True)
    run()
    ctx.prof_enable(False)
    return [k["name"].split()[0] for k in ctx.prof_report()["kernels"]]


def test_the_switch_fixes_the_tile(tiled):
    c, tile = tiled
    x, w = L.Mat(c, np.ones((3, 5), np.float32)), L.Mat(c, np.ones((5, 7), np.float32))
    assert names(c, lambda: L.forward(c, x, w)) == [f"linear_act_t{tile}"]
    dw = L.Mat(c, shape=(5, 7))
    assert names(c, lambda: L.backward(c, L.Mat(c, np.ones((3, 7), np.float32)), w, x=x, dw=dw)) == \
        [f"linear_act_backward_t{tile}"]


# shapes that the kernels for few rows and for small backwards take: 1 .. 16 rows, widths around 16, 64 and 256
# columns and below 4, and past 16 columns for each CU (blocks of 2 to 16 groups), k of one wave's step, of several,
# and split
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 256), (2, 17, 100), (3, 3, 2000), (4, 258, 4100), (4, 4096, 700),
                                   (1, 70, 9000), (5, 64, 65), (9, 255, 63), (16, 256, 128), (16, 1030, 70),
                                   (17, 130, 40), (12, 2, 300),
                                   (2, 5001, 300), (3, 9000, 70), (1, 17003, 257), (4, 40000, 33), (5, 5001, 130),
                                   (6, 33, 3100), (7, 8200, 40), (8, 66000, 17), (8, 30, 5000), (8, 4100, 1100)])
def test_few_rows(ctx, m, n, k):
    L.test_forward(ctx, m, n, k)
    L.test_backward(ctx, m, n, k)


def test_which_kernels_take_what(ctx):
    def fwd(m, n, k):
        x, w = L.Mat(ctx, np.ones((m, k), np.float32)), L.Mat(ctx, np.ones((k, n), np.float32))
        return names(ctx, lambda: L.forward(ctx, x, w))

    def bwd(m, n, k, act):
        one = lambda *s: L.Mat(ctx, np.ones(s, np.float32))  # noqa: E731
        return names(ctx, lambda: L.backward(ctx, one(m, n), one(k, n), act, z=one(m, n) if act != "none" else None,
                                             x=one(m, k), dx=one(m, k), dw=one(k, n), db=one(1, n)))

    assert fwd(8, 300, 300) == ["linear_act_rows"] and fwd(9, 300, 300) == ["linear_act_t64"]
    assert bwd(64, 128, 128, "gelu") == ["linear_act_backward_inside_t64"]
    assert bwd(4, 128, 128, "gelu") == ["linear_act_backward_inside_rows"]
    assert bwd(16, 128, 128, "none") == ["linear_act_backward_inside_rows"]
    assert bwd(16, 128, 128, "gelu") == ["linear_act_backward_inside_t64"]
    assert set(bwd(16, 2048, 2048, "gelu")) == {"linear_act_slope", "linear_act_backward_rows"}
    assert set(bwd(600, 512, 512, "none")) == {"linear_act_slope", "linear_act_backward_t64"}


@pytest.mark.parametrize("m,n,k,act", [(3, 40, 70, "silu"), (12, 40, 70, "none"), (12, 600, 4100, "gelu"),
                                       (100, 60, 80, "gelu_tanh"), (700, 130, 257, "silu")])
@pytest.mark.parametrize("want", ["dx", "dw", "db", "dx dw", "dw db", "dx db", ""])
def test_each_output_alone(ctx, m, n, k, act, want):
    rng = np.random.default_rng(m + n + k)
    x, w, b, dy = L.data(rng, m, n, k)
    z = (x.astype(np.float64) @ w + b).astype(np.float32)
    dz = dy * L.act64(act, z.astype(np.float64))[1]
    dztol = np.abs(dy) * L.slope_tol(z.astype(np.float64)) * (act != "none") + L.U * np.abs(dz)
    out = {}
    if "dx" in want:
        out["dx"] = L.Mat(ctx, shape=(m, k))
    if "dw" in want:
        out["dw"] = L.Mat(ctx, shape=(k, n))
    if "db" in want:
        out["db"] = L.Mat(ctx, shape=(1, n))
    L.backward(ctx, L.Mat(ctx, dy), L.Mat(ctx, w), act, z=L.Mat(ctx, z) if act != "none" else None,
               x=L.Mat(ctx, x) if "dw" in want else None, **out)
    aw, ax = np.abs(w).astype(np.float64), np.abs(x).astype(np.float64)
    if "dx" in want:
        L.close(out["dx"].get(), dz @ w.T.astype(np.float64), L.product_tol(np.abs(dz) @ aw.T, n) + dztol @ aw.T, "dx")
    if "dw" in want:
        L.close(out["dw"].get(), x.T.astype(np.float64) @ dz, L.product_tol(ax.T @ np.abs(dz), m) + ax.T @ dztol, "dw")
    if "db" in want:
        # at most rows / 16 additions of a thread, 16 runs, and the rounding of blocks of 64
        tol = L.U * (m / 16 + 64) * np.abs(dz).sum(0, keepdims=True) + dztol.sum(0, keepdims=True)
        L.close(out["db"].get(), dz.sum(0, keepdims=True), tol, "db")


def test_columns_of_one_matrix(ctx):
    """Operands that are columns of one wide matrix: nothing but y's, or dx's, columns changes."""
    m, n, k = 70, 40, 40
    rng = np.random.default_rng(3)
    x, w, b, r = L.data(rng, m, n, k)
    want = L.forward(ctx, L.Mat(ctx, x), L.Mat(ctx, w), "silu", L.Mat(ctx, b), L.Mat(ctx, r)).get()
    wide = np.full((m, 200), L.SENTINEL, np.float32)
    wide[:, 10:10 + k], wide[:, 110:110 + n] = x, r
    buf = ctx.upload(wide)
    at = lambda c: buf.ptr + 4 * c  # noqa: E731
    W, B = L.Mat(ctx, w), L.Mat(ctx, b)
    e = _lib.LinearEpilogue(act=_lib.ACT_SILU, bias=B.ptr, residual=at(110), ldr=200)
    _lib.call("orca_hip_linear_act", ctx.handle, m, n, k, at(10), 200, W.ptr, n, at(60), 200, ctypes.byref(e))
    got = buf.download().reshape(m, 200)
    np.testing.assert_array_equal(got[:, 60:60 + n], want)
    got[:, 60:60 + n] = L.SENTINEL
    np.testing.assert_array_equal(got, wide)
    with pytest.raises(ValueError, match="overlaps"):
        _lib.call("orca_hip_linear_act", ctx.handle, m, n, k, at(10), 200, W.ptr, n, at(49), 200, ctypes.byref(e))
    with pytest.raises(ValueError, match="overlaps"):
        _lib.call("orca_hip_linear_act", ctx.handle, m, n, k, at(10), 200, W.ptr, n, at(71), 200, ctypes.byref(e))


def test_buffers_that_are_too_small(ctx):
    """A buffer holds at least what was asked for, in the allocator's granules: the calls here go past those."""
    x, w, y = (L.Mat(ctx, np.ones((8, 8), np.float32)) for _ in range(3))
    X, W, Y = (L.Mat(ctx, np.ones((128, 128), np.float32)) for _ in range(3))
    small = ctx.alloc(64)
    with pytest.raises(ValueError, match="Shape mismatch"):
        _lib.call("orca_hip_linear_act", ctx.handle, 8, 80, 8, x.ptr, 8, w.ptr, 80, y.ptr, 80, None)
    with pytest.raises(ValueError, match="Shape mismatch"):
        e = _lib.LinearEpilogue(y8=small.ptr)
        _lib.call("orca_hip_linear_act", ctx.handle, 128, 128, 128, X.ptr, 128, W.ptr, 128, Y.ptr, 128,
                  ctypes.byref(e))
    with pytest.raises(ValueError, match="Shape mismatch"):
        _lib.call("orca_hip_act8_pack", ctx.handle, X.ptr, 128, 128, 128, small.ptr)
    with pytest.raises(ValueError, match="Shape mismatch"):
        _lib.call("orca_hip_act8_unpack", ctx.handle, small.ptr, 128, 128, _lib.F32, Y.ptr, 128)


def test_matrices_past_4_gib(ctx):
    """A weight of 4.3 GiB, its gradient and a checkpoint of 1.1 GiB: the last rows and columns come
    from and go to their own place."""
    n = k = 34000
    rows = {0: 1.0, 1: -2.0, k // 2: 0.5, k - 2: 3.0, k - 1: 4.0}  # k: the value of W's row
    w = ctx.alloc(4 * n * k)
    ctx.fill(w, 0.0, n * k)
    for r, v in rows.items():
        line = np.full(n, v, np.float32)
        line[-1] += 0.25
        _lib.call("orca_hip_h2d", ctx.handle, w.ptr + 4 * n * r, line.ctypes.data_as(ctypes.c_void_p), line.nbytes)
    rng = np.random.default_rng(1)
    for m in (2, 7):
        x = np.zeros((m, k), np.float32)
        x[:, list(rows)] = rng.integers(-4, 5, (m, len(rows)))
        vals = np.array(list(rows.values()))
        want = x[:, list(rows)].astype(np.float64) @ vals
        X = L.Mat(ctx, x)
        y = L.Mat(ctx, shape=(m, n))
        _lib.call("orca_hip_linear_act", ctx.handle, m, n, k, X.ptr, k, w.ptr, n, y.ptr, n, None)
        got = y.get()
        np.testing.assert_array_equal(got[:, :-1], np.repeat(want[:, None], n - 1, 1).astype(np.float32))
        np.testing.assert_array_equal(got[:, -1], x[:, list(rows)].astype(np.float64) @ (vals + 0.25))
        dy = np.zeros((m, n), np.float32)
        dy[:, [0, n - 1]] = rng.integers(-4, 5, (m, 2))
        DY, dx = L.Mat(ctx, dy), L.Mat(ctx, shape=(m, k))
        dw = ctx.alloc(4 * n * k)
        ctx.fill(dw, 7.0, n * k)
        s = _lib.LinearSaved(x=X.ptr, ldx=k)
        _lib.call("orca_hip_linear_act_backward", ctx.handle, m, n, k, DY.ptr, n, w.ptr, n, ctypes.byref(s), dx.ptr, k,
                  dw.ptr, n, None)
        got = dx.get()
        for r, v in rows.items():
            np.testing.assert_array_equal(got[:, r], dy[:, 0] * v + dy[:, -1] * (v + 0.25))
        want_dw = x.T.astype(np.float64) @ dy
        for r in list(rows) + [17, k - 5]:
            line = np.empty(n, np.float32)
            _lib.call("orca_hip_d2h", ctx.handle, line.ctypes.data_as(ctypes.c_void_p), dw.ptr + 4 * n * r, line.nbytes)
            np.testing.assert_array_equal(line, want_dw[r])
    q = ctx.alloc(L.layout(k, n)[3])
    _lib.call("orca_hip_act8_pack", ctx.handle, w.ptr, k, n, n, q.ptr)
    ctx.fill(dw, 7.0, n * k)
    _lib.call("orca_hip_act8_unpack", ctx.handle, q.ptr, k, n, _lib.F32, dw.ptr, n)
    for r in list(rows) + [5]:
        line = np.empty(n, np.float32)
        _lib.call("orca_hip_d2h", ctx.handle, line.ctypes.data_as(ctypes.c_void_p), dw.ptr + 4 * n * r, line.nbytes)
        v = rows.get(r, 0.0)
        np.testing.assert_array_equal(line[:-1], v)
        assert line[-1] == (v + 0.25 if r in rows else 0.0)
    # as the weight gradient's operand: its rows are the k values
    dy = np.zeros((k, 3), np.float32)
    dy[list(rows)] = rng.integers(-4, 5, (len(rows), 3))
    out = L.Mat(ctx, shape=(n, 3))
    DY = L.Mat(ctx, dy)
    s = _lib.LinearSaved(x8=q.ptr)
    _lib.call("orca_hip_linear_act_backward", ctx.handle, k, 3, n, DY.ptr, 3, None, 3, ctypes.byref(s), None, 0, out.ptr, 3,
              None)
    vals = np.array(list(rows.values()))
    got = out.get()
    np.testing.assert_array_equal(got[:-1], np.repeat((vals @ dy[list(rows)].astype(np.float64))[None], n - 1, 0))
    np.testing.assert_array_equal(got[-1], (vals + 0.25) @ dy[list(rows)].astype(np.float64))


def test_tall_and_wide(ctx):
    """Many rows against few columns, and the other way round, where k or an output is long."""
    rng = np.random.default_rng(2)
    for m, n, k in ((100000, 3, 5), (3, 100000, 5), (30, 70000, 4), (50000, 20, 20)):
        x, w, b, r = L.data(rng, m, n, k)
        z64 = x.astype(np.float64) @ w + b
        ztol = L.product_tol(np.abs(x).astype(np.float64) @ np.abs(w) + np.abs(b), k)
        y = L.forward(ctx, L.Mat(ctx, x), L.Mat(ctx, w), "silu", L.Mat(ctx, b)).get()
        L.close(y, L.act64("silu", z64)[0], L.act_tol(z64, ztol) + 2 * L.U * np.abs(z64), "y")
        dx, dw, db = L.Mat(ctx, shape=(m, k)), L.Mat(ctx, shape=(k, n)), L.Mat(ctx, shape=(1, n))
        L.backward(ctx, L.Mat(ctx, r), L.Mat(ctx, w), x=L.Mat(ctx, x), dx=dx, dw=dw, db=db)
        r64 = r.astype(np.float64)
        L.close(dx.get(), r64 @ w.T, L.product_tol(np.abs(r64) @ np.abs(w.T), n), "dx")
        # up to 256 splits, added in order
        L.close(dw.get(), x.T.astype(np.float64) @ r64,
                L.product_tol(np.abs(x.T).astype(np.float64) @ np.abs(r64), m) + 256 * L.U * (np.abs(x.T) @ np.abs(r64)), "dw")
        L.close(db.get(), r64.sum(0, keepdims=True), L.U * (m / 512 + 64) * np.abs(r64).sum(0, keepdims=True), "db")


def test_tiny_magnitudes(ctx):
    """Below 2^-100 a value keeps fewer bits, below 2^-126 none: the error of a product with 1 is at most
    2^-126, and there is no NaN."""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((64, 64)) * 2.0 ** rng.integers(-149, -95, (64, 64))).astype(np.float32)
    y = L.forward(ctx, L.Mat(ctx, x), L.Mat(ctx, np.eye(64, dtype=np.float32))).get()
    assert (np.abs(y.astype(np.float64) - x) <= 2.0 ** -125).all()
    fine = np.abs(x) >= 2.0 ** -100
    np.testing.assert_array_equal(y[fine], x[fine])


@pytest.mark.parametrize("m,n,k", [(1, (1 << 25) + 5, 1), (3, 17000003, 2), ((1 << 25) + 5, 1, 1), (40000000, 2, 3),
                                   (20, 17000001, 1), (1, 2, 17000001)])
def test_the_longest_sizes(ctx, m, n, k):
    """Past 65535 blocks of 256 columns, past the few rows' longest rows, and millions of rows: small whole numbers, so
    exact (the checkpoint too: codes of up to 7 bits with steps of powers of two)."""
    x = (np.arange(m * k, dtype=np.int64) % 7 - 3).astype(np.float32).reshape(m, k)
    w = (np.arange(k * n, dtype=np.int64) % 5 - 2).astype(np.float32).reshape(k, n)
    want = sum(x[:, i:i + 1] * w[i:i + 1] for i in range(k)) if k < 10 else x @ w
    if k >= 10:  # by sums that stay whole numbers below 2^24
        want = np.add.reduce((x[0][:, None] * w).astype(np.float64), axis=0)[None].astype(np.float32)
    X, W, y8 = L.Mat(ctx, x), L.Mat(ctx, w), L.Packed(ctx, m, n)
    np.testing.assert_array_equal(L.forward(ctx, X, W, y8=y8).get(), want)
    small = np.abs(want).max() < 64
    back = L.Mat(ctx, shape=(m, n))
    _lib.call("orca_hip_act8_unpack", ctx.handle, y8.ptr, m, n, _lib.F32, back.ptr, n)
    if small:
        np.testing.assert_array_equal(back.get(), want)
    z = (np.arange(m * n, dtype=np.int64) % 3 - 1).astype(np.float32).reshape(m, n)
    dy = (np.arange(m * n, dtype=np.int64) % 11 - 5).astype(np.float32).reshape(m, n)
    g = dy * (z > 0)
    dx, dw, db = L.Mat(ctx, shape=(m, k)), L.Mat(ctx, shape=(k, n)), L.Mat(ctx, shape=(1, n))
    L.backward(ctx, L.Mat(ctx, dy), W, "relu", z=L.Mat(ctx, z), x=X, dx=dx, dw=dw, db=db)
    g64 = g.astype(np.float64)
    for what, got, exact, size in (("db", db, g64.sum(0, keepdims=True), np.abs(g64).sum(0).max()),
                                   ("dx", dx, g64 @ w.T.astype(np.float64), 10 * n),
                                   ("dw", dw, x.T.astype(np.float64) @ g64, 15 * m)):
        got = got.get()
        if size < 1 << 24:
            np.testing.assert_array_equal(got, exact, err_msg=what)
        else:
            # fp32 sums of whole numbers: runs of at most 2^15 terms and fewer than 2^12 runs a sum, each addition off by half a
            # step of a partial sum, which stays below `size`; steps of runs are exact below 2^24
            tol = 2.0 ** -24 * (1 << 12) * np.abs(exact) + 2.0 ** -24 * size * 600
            assert (np.abs(got - exact) <= tol).all(), what
