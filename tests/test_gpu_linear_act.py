"""The Linear with activation and residual (orca_hip_linear_act, its backward) and the 8-bit
activation checkpoints against a plain implementation in 64 bits.

Tolerances of a product.  Its terms are taken to below 2^-23 of each product (three left out, each
centred on zero), and fp32 sums run over 6 * ceil(K / 16) matrix instructions and at most 64 splits:
with the roundings independent, the error's standard deviation is below 2^-25 * sqrt(steps) of the
largest running sum, which is at most S = sum |x| |w|; running sums are far smaller than S as soon as
signs mix.  2^-24 * (8 + 2 sqrt(steps)) * S is four of these deviations and the constant's few roundings
(bias, the instruction's own sums, the terms left out)."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
from scipy.special import erfc

from orcaml_amd import _lib

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
U = 2.0 ** -24  # half a step of fp32, relative


# ---------------------------------------------------------------- plain, in 64 bits
def act64(kind, z):
    """(act(z), act'(z))"""
    with np.errstate(over="ignore", under="ignore"):
        if kind == "relu":
            return np.where(z > 0, z, 0.0), (z > 0) * 1.0
        if kind == "gelu":
            phi = 0.5 * erfc(-z / math.sqrt(2))
            return z * phi, phi + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        if kind == "gelu_tanh":
            c = math.sqrt(2 / math.pi)
            t = np.tanh(c * (z + 0.044715 * z ** 3))
            return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
        if kind == "silu":
            s = 1 / (1 + np.exp(-z))
            return z * s, s * (1 + z * (1 - s))
    return z, np.ones_like(z)


def steps(k):
    return 6 * math.ceil(k / 16) + 64


def product_tol(s, k):
    return U * (8 + 2 * math.sqrt(steps(k))) * s


# Slopes of the activations lie within [-0.2, 1.2] and change by at most 1.1 per unit of z.  The
# functions themselves are a few roundings of values of the order of 1 + |z|: 2^-20 (1 + |z|).
def act_tol(z, ztol):
    return 1.2 * ztol + 2.0 ** -20 * np.abs(z) + 1e-37


def slope_tol(z):
    return 2.0 ** -20 * (1 + np.abs(z)) * (np.abs(z) < 30) + 2.0 ** -22


def layout(rows, cols):
    groups, ld = -(-cols // 32), -(-rows // 16) * 16
    at = -(-rows * cols // 16) * 16
    return groups, ld, at, at + groups * ld


def pack64(x):
    """(codes [rows][cols] int, step bytes [rows][groups]) from the definition."""
    rows, cols = x.shape
    groups = -(-cols // 32)
    codes, bytes_ = np.zeros((rows, cols), np.int64), np.zeros((rows, groups), np.int64)
    for g in range(groups):
        part = x[:, 32 * g:32 * g + 32].astype(np.float64)
        for r in range(rows):
            if not np.isfinite(part[r]).all():
                bytes_[r, g] = 255
                continue
            top = np.abs(part[r]).max()
            b = 7 if top == 0 else max(7, int(math.floor(math.log2(top))) + 125)
            while b < 254 and np.abs(np.rint(part[r] * 2.0 ** (133 - b))).max() > 127:
                b += 1
            while b > 7 and np.abs(np.rint(part[r] * 2.0 ** (134 - b))).max() <= 127:
                b -= 1
            bytes_[r, g] = b
            codes[r, 32 * g:32 * g + 32][:part.shape[1]] = np.clip(np.rint(part[r] * 2.0 ** (133 - b)), -127, 127)
    return codes, bytes_


def read_packed(buf, rows, cols):
    groups, ld, at, _ = layout(rows, cols)
    codes = buf[:rows * cols].view(np.int8).reshape(rows, cols).astype(np.int64)
    return codes, buf[at:].reshape(groups, ld)[:, :rows].T.astype(np.int64)


def value64(codes, bytes_):
    step = np.where(bytes_ == 255, np.nan, 2.0 ** (bytes_.astype(np.float64) - 133))
    return codes * np.repeat(step, 32, axis=1)[:, :codes.shape[1]]


def write_packed(codes, bytes_):
    rows, cols = codes.shape
    groups, ld, at, size = layout(rows, cols)
    buf = np.full(size, 0xA5, np.uint8)  # what lies between and behind the rows means nothing
    buf[:rows * cols] = codes.astype(np.int8).reshape(-1).view(np.uint8)
    buf[at:].reshape(groups, ld)[:, :rows] = bytes_.T.astype(np.uint8)
    return buf


# ---------------------------------------------------------------- device matrices
SENTINEL = np.float32(-7.25e11)


class Mat:
    """A matrix in a buffer with a leading dimension, an offset of floats and sentinels around it."""

    def __init__(self, ctx, data=None, shape=None, pad=0, off=0):
        self.rows, self.cols = data.shape if data is not None else shape
        self.ld, self.off = self.cols + pad, off
        host = np.full(off + self.rows * self.ld + 64, SENTINEL, np.float32)
        if data is not None:
            self._view(host)[:] = data
        self.host, self.buf = host, ctx.upload(host)

    def _view(self, host):
        return host[self.off:self.off + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    @property
    def ptr(self):
        return self.buf.ptr + 4 * self.off

    def get(self):
        """The matrix, after a look at what lies around it."""
        host = self.buf.download()
        out = self._view(host).copy()
        self._view(host)[:] = SENTINEL
        assert (host == SENTINEL).all(), "written outside the matrix"
        return out


class Packed:
    def __init__(self, ctx, rows, cols, data=None):
        self.rows, self.cols, self.size = rows, cols, layout(rows, cols)[3]
        self.buf = ctx.upload(data if data is not None else np.full(self.size, 0x5A, np.uint8))

    @property
    def ptr(self):
        return self.buf.ptr

    def get(self):
        return read_packed(self.buf.download(np.uint8, self.size), self.rows, self.cols)


def forward(ctx, x, w, act="none", bias=None, residual=None, pre=None, pre8=None, y8=None, y=None, pad=0):
    y = y or Mat(ctx, shape=(x.rows, w.cols), pad=pad)
    e = _lib.LinearEpilogue(act=ACTS.index(act), bias=bias.ptr if bias else None,
                            residual=residual.ptr if residual else None, ldr=residual.ld if residual else 0,
                            pre=pre.ptr if pre else None, ldpre=pre.ld if pre else 0, pre8=pre8.ptr if pre8 else None,
                            y8=y8.ptr if y8 else None)
    _lib.call("orca_hip_linear_act", ctx.handle, x.rows, w.cols, x.cols, x.ptr, x.ld, w.ptr, w.ld, y.ptr, y.ld,
              ctypes.byref(e))
    return y


def backward(ctx, dy, w, act="none", z=None, z8=None, x=None, x8=None, add=None, dx=None, dw=None, db=None):
    s = _lib.LinearSaved(act=ACTS.index(act), z=z.ptr if z else None, ldz=z.ld if z else 0, z8=z8.ptr if z8 else None,
                         x=x.ptr if x else None, ldx=x.ld if x else 0, x8=x8.ptr if x8 else None,
                         dx_add=add.ptr if add else None, ldadd=add.ld if add else 0)
    k = w.rows
    _lib.call("orca_hip_linear_act_backward", ctx.handle, dy.rows, dy.cols, k, dy.ptr, dy.ld, w.ptr, w.ld,
              ctypes.byref(s), dx.ptr if dx else None, dx.ld if dx else 0, dw.ptr if dw else None,
              dw.ld if dw else 0, db.ptr if db else None)


def close(got, want, tol, what):
    err = np.abs(got.astype(np.float64) - want)
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(err / np.maximum(tol, 1e-300)):.3g} " \
                          f"of the tolerance at {np.unravel_index(np.argmax(bad), bad.shape)}"


def data(rng, m, n, k):
    x = (rng.standard_normal((m, k)) * np.exp(rng.standard_normal((1, k)) * 0.5)).astype(np.float32)
    w = (rng.uniform(-1, 1, (k, n)) / math.sqrt(max(k, 1))).astype(np.float32)
    return x, w, (rng.standard_normal((1, n)) * 0.1).astype(np.float32), rng.standard_normal((m, n)).astype(np.float32)


# rows, columns and k: one of each, around the tiles, the stages and the splits, odd ones, long k
SHAPES = [(1, 1, 1), (1, 7, 3), (3, 5, 17), (1, 300, 515), (2, 64, 4096), (15, 33, 31), (16, 32, 16), (31, 127, 129),
          (33, 65, 40), (64, 128, 784), (65, 257, 100), (100, 36, 1003), (129, 130, 15), (256, 256, 256),
          (257, 300, 333), (128, 1000, 64), (700, 10, 130), (513, 511, 255), (40, 40, 9000)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward(ctx, m, n, k):
    rng = np.random.default_rng(m * 7919 + n * 31 + k)
    x, w, b, r = data(rng, m, n, k)
    z64 = x.astype(np.float64) @ w.astype(np.float64) + b
    s = np.abs(x).astype(np.float64) @ np.abs(w) + np.abs(b)
    ztol = product_tol(s, k)
    dx, dw, db, dr = Mat(ctx, x), Mat(ctx, w), Mat(ctx, b), Mat(ctx, r)
    for i, act in enumerate(ACTS):
        print(f"forward {m}x{n}x{k} {act}", flush=True)
        pre, z8, y8 = Mat(ctx, shape=(m, n)), Packed(ctx, m, n), Packed(ctx, m, n)
        res = dr if i % 2 == 0 else None
        y = forward(ctx, dx, dw, act, db, res, pre, z8, y8).get()
        z = pre.get()
        close(z, z64, ztol, f"z {act}")
        y64 = act64(act, z64)[0] + (r if res else 0.0)
        close(y, y64, act_tol(z64, ztol) + 2 * U * np.abs(y64), f"y {act}")
        for name, got, of in (("z8", z8.get(), z), ("y8", y8.get(), y)):  # what packing these very values gives
            codes, bytes_ = pack64(of)
            np.testing.assert_array_equal(got[1], bytes_, err_msg=f"{name} bytes {act}")
            np.testing.assert_array_equal(got[0], codes, err_msg=f"{name} codes {act}")
    plain = forward(ctx, dx, dw).get()  # no epilogue at all
    close(plain, z64 - b, ztol, "plain product")


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_backward(ctx, m, n, k):
    rng = np.random.default_rng(m * 7919 + n * 31 + k + 1)
    x, w, b, _ = data(rng, m, n, k)
    dy = rng.standard_normal((m, n)).astype(np.float32)
    add = rng.standard_normal((m, k)).astype(np.float32)
    z = (x.astype(np.float64) @ w + b).astype(np.float32)
    z[rng.random((m, n)) < 0.05] = 0.0
    xc, xb = pack64(x)
    zc, zb = pack64(z)
    devs = dict(dy=Mat(ctx, dy), w=Mat(ctx, w))
    mx, mz, madd = Mat(ctx, x), Mat(ctx, z), Mat(ctx, add)
    mx8, mz8 = Packed(ctx, m, k, write_packed(xc, xb)), Packed(ctx, m, n, write_packed(zc, zb))
    for i, act in enumerate(ACTS):
        for kept in ("fp32", "8bit"):
            print(f"backward {m}x{n}x{k} {act} {kept}", flush=True)
            x64, z64 = (x.astype(np.float64), z.astype(np.float64)) if kept == "fp32" else (value64(xc, xb), value64(zc, zb))
            slope = act64(act, z64)[1]
            dz = dy * slope
            dztol = np.abs(dy) * slope_tol(z64) * (act not in ("none", "relu")) + U * np.abs(dz)
            with_add = i % 2 == 0
            dx, dw, db = Mat(ctx, shape=(m, k)), Mat(ctx, shape=(k, n)), Mat(ctx, shape=(1, n))
            saved = dict(x=mx, z=mz) if kept == "fp32" else dict(x8=mx8, z8=mz8)
            if act == "none":
                saved.pop("z", None), saved.pop("z8", None)
            backward(ctx, devs["dy"], devs["w"], act, add=madd if with_add else None, dx=dx, dw=dw, db=db, **saved)
            aw, ax = np.abs(w).astype(np.float64), np.abs(x64)
            want = dz @ w.T.astype(np.float64) + (add if with_add else 0.0)
            close(dx.get(), want, product_tol(np.abs(dz) @ aw.T, n) + dztol @ aw.T + 2 * U * np.abs(want), f"dx {act} {kept}")
            close(dw.get(), x64.T @ dz, product_tol(ax.T @ np.abs(dz), m) + ax.T @ dztol, f"dw {act} {kept}")
            # sums of 16 rows, of 4, of at most ceil(blocks / 8) blocks and of 8 runs
            adds = 16 + 4 + math.ceil(m / 512) + 8
            close(db.get(), dz.sum(0, keepdims=True), U * adds * np.abs(dz).sum(0, keepdims=True)
                  + dztol.sum(0, keepdims=True), f"db {act} {kept}")


def test_leading_dimensions_and_alignment(ctx):
    """Padded rows, and matrices that start at any float: nothing outside them is read into a result
    or written."""
    m, n, k = 130, 70, 50
    rng = np.random.default_rng(5)
    x, w, b, r = data(rng, m, n, k)
    dy, add = rng.standard_normal((m, n)).astype(np.float32), rng.standard_normal((m, k)).astype(np.float32)
    base = {}
    for off in range(4):
        for pad in (0, 1, 5):
            kw = dict(pad=pad, off=off)
            X, W, B, R = Mat(ctx, x, **kw), Mat(ctx, w, **kw), Mat(ctx, b, off=off), Mat(ctx, r, **kw)
            y, pre = Mat(ctx, shape=(m, n), **kw), Mat(ctx, shape=(m, n), **kw)
            forward(ctx, X, W, "silu", B, R, pre, y=y)
            dx, dw, db = Mat(ctx, shape=(m, k), **kw), Mat(ctx, shape=(k, n), **kw), Mat(ctx, shape=(1, n), off=off)
            backward(ctx, Mat(ctx, dy, **kw), W, "silu", z=pre, x=X, add=Mat(ctx, add, **kw), dx=dx, dw=dw, db=db)
            for name, t in (("y", y), ("pre", pre), ("dx", dx), ("dw", dw), ("db", db)):
                got = t.get()
                np.testing.assert_array_equal(got, base.setdefault(name, got), err_msg=f"{name} off {off} pad {pad}")


def test_in_place_residual_and_gradient(ctx):
    m, n, k = 200, 96, 96
    rng = np.random.default_rng(6)
    x, w, b, r = data(rng, m, n, k)
    X, W, B = Mat(ctx, x), Mat(ctx, w), Mat(ctx, b)
    want = forward(ctx, X, W, "gelu", B, Mat(ctx, r, pad=3)).get()
    y = Mat(ctx, r, pad=3)
    np.testing.assert_array_equal(forward(ctx, X, W, "gelu", B, y, y=y).get(), want)
    DY = Mat(ctx, r)
    dx = Mat(ctx, shape=(m, k))
    backward(ctx, DY, W, add=X, x=X, dx=dx)
    acc = Mat(ctx, x)
    backward(ctx, DY, W, add=acc, x=X, dx=acc)
    np.testing.assert_array_equal(acc.get(), dx.get())
    both = Mat(ctx, shape=(m, k))  # y = act(x w) + x: the residual's gradient is dy itself
    backward(ctx, DY, W, add=DY, dx=both)
    close(both.get(), r + r.astype(np.float64) @ w.T, product_tol(np.abs(r) @ np.abs(w.T).astype(np.float64), n) + U * 8,
          "dx + dy")


@pytest.mark.parametrize("m,n,k", [(0, 5, 7), (5, 0, 7), (5, 7, 0), (0, 0, 0), (1, 0, 0), (0, 3, 0), (70, 40, 0)])
def test_empty_sizes(ctx, m, n, k):
    rng = np.random.default_rng(7)
    x, w, b, r = data(rng, m, n, k)
    pre = Mat(ctx, shape=(m, n))
    y = forward(ctx, Mat(ctx, x), Mat(ctx, w), "silu", Mat(ctx, b), Mat(ctx, r), pre).get()
    z64 = np.broadcast_to(b.astype(np.float64), (m, n))
    close(y, act64("silu", z64)[0] + r, act_tol(z64, 0.0) + 4 * U * (1 + np.abs(r)), "y")
    np.testing.assert_array_equal(pre.get(), np.broadcast_to(b, (m, n)))
    add = rng.standard_normal((m, k)).astype(np.float32)
    dx, dw, db = Mat(ctx, shape=(m, k)), Mat(ctx, shape=(k, n)), Mat(ctx, shape=(1, n))
    backward(ctx, Mat(ctx, r), Mat(ctx, w), "silu", z=pre, x=Mat(ctx, x), add=Mat(ctx, add), dx=dx, dw=dw, db=db)
    if n == 0:
        np.testing.assert_array_equal(dx.get(), add)
    if m == 0:
        assert not dw.get().any() and not db.get().any()


def test_split_products_are_exact_where_fp32_is(ctx):
    """One term per element: each product of an fp32 value of any bits with a power of two comes back
    as it is, so no bit of a value is lost in its three terms."""
    rng = np.random.default_rng(8)
    m, k = 300, 200
    bits = rng.integers(0, 1 << 32, (m, k), dtype=np.uint64).astype(np.uint32)
    x = bits.view(np.float32).copy()
    # exponents that leave the terms and the product normal
    x[~np.isfinite(x) | (np.abs(x) < 2.0 ** -90) | (np.abs(x) > 2.0 ** 126)] = 1.2345678
    x[0, :8] = np.float32(2.0) ** 127 * np.float32(2 - 2.0 ** -23)  # the largest: rounds up in bf16
    w = np.zeros((k, k), np.float32)
    w[np.arange(k), rng.permutation(k)] = 1.0
    y = forward(ctx, Mat(ctx, x), Mat(ctx, w)).get()
    np.testing.assert_array_equal(y, x @ w)
    half = np.where(np.abs(x) > 2.0 ** 100, np.float32(1), x)
    w2 = (w * 0.5 ** rng.integers(0, 4, (k, 1))).astype(np.float32)
    dx, dw = Mat(ctx, shape=(m, k)), Mat(ctx, shape=(k, k))
    backward(ctx, Mat(ctx, half), Mat(ctx, w2), x=Mat(ctx, np.eye(m, k, dtype=np.float32)), dx=dx, dw=dw)
    np.testing.assert_array_equal(dx.get(), half @ w2.T)
    np.testing.assert_array_equal(dw.get(), half[:k, :])


def test_integers_are_exact(ctx):
    rng = np.random.default_rng(9)
    for m, n, k in [(64, 64, 64), (257, 129, 77), (9, 500, 1030)]:
        x = rng.integers(-2000, 2000, (m, k)).astype(np.float32)
        w = rng.integers(-8, 8, (k, n)).astype(np.float32)
        y = forward(ctx, Mat(ctx, x), Mat(ctx, w)).get()
        np.testing.assert_array_equal(y, (x.astype(np.int64) @ w.astype(np.int64)).astype(np.float32))


@pytest.mark.parametrize("m,n,k", [(4, 40, 48), (150, 140, 100), (70, 70, 3000)])
def test_infinities_and_nan_come_out_as_from_fp32(ctx, m, n, k):
    rng = np.random.default_rng(10)
    x, w, _, _ = data(rng, m, n, k)
    x[1, 3], x[2, 5], x[3, 7], x[3, 8] = np.inf, np.nan, -np.inf, np.inf
    x[0, 4] = np.uint32(0x7f800001).view(np.float32)  # a NaN whose upper half is an infinity's
    w[3, 0], w[3, 1], w[3, 2] = 1.0, -2.0, 0.0  # inf times values without lower terms, and times zero
    w[9, 5], w[10, 6] = np.inf, np.nan
    x[1, 9] = 0.0
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64)
        dy = x
        dxw = dy.astype(np.float64) @ np.ones((k, n))
    y = forward(ctx, Mat(ctx, x), Mat(ctx, w)).get()
    np.testing.assert_array_equal(np.isnan(y), np.isnan(want))
    inf = np.isinf(want)
    assert inf.any()
    np.testing.assert_array_equal(y[inf], want[inf].astype(np.float32))
    fine = np.isfinite(want)
    s = np.abs(np.where(np.isfinite(x), x, 0)).astype(np.float64) @ np.abs(np.where(np.isfinite(w), w, 0))
    close(np.where(fine, y, 0), np.where(fine, want, 0), product_tol(s, k) + 1e-30, "finite part")
    dx = Mat(ctx, shape=(m, n))
    backward(ctx, Mat(ctx, x), Mat(ctx, np.ones((n, k), np.float32)), dx=dx)  # every row with an infinity or NaN
    got = dx.get()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(dxw))
    np.testing.assert_array_equal(got[np.isinf(dxw)], dxw[np.isinf(dxw)].astype(np.float32))


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (17, 100), (64, 1000), (16, 4096), (33, 257),
                                       (1000, 7)])
def test_pack_and_unpack(ctx, rows, cols):
    rng = np.random.default_rng(rows * 5003 + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, cols)) * 3)).astype(np.float32)
    x.reshape(-1)[::37] = 0.0
    x.reshape(-1)[5::41] = -0.0
    x[rows // 2, :min(cols, 32)] = 0.0  # a group of zeros
    flat = x.reshape(-1)
    for i, v in enumerate([1.0, 127.4 / 64, 127.5 / 64, 127.6 / 64, -2.0, 3.4028234e38, 127.5 * 2.0 ** 121, 1e-45,
                           2.0 ** -120, 2.0 ** -126, 2.0 ** -127]):
        if 32 * i + 3 < flat.size:
            flat[32 * i + 3] = v
    for pad, off in ((0, 0), (3, 1)):
        p = Packed(ctx, rows, cols)
        X = Mat(ctx, x, pad=pad, off=off)
        _lib.call("orca_hip_act8_pack", ctx.handle, X.ptr, rows, cols, X.ld, p.ptr)
        codes, bytes_ = p.get()
        want = pack64(x)
        np.testing.assert_array_equal(bytes_, want[1])
        np.testing.assert_array_equal(codes, want[0])
        value = value64(*want)
        top = np.abs(x.astype(np.float64))
        step = np.repeat(2.0 ** (want[1] - 133.0), 32, axis=1)[:, :cols]
        clipped = top > 127.5 * step  # at the very end of the range
        assert (np.abs(value - x)[~clipped] <= step[~clipped] / 2).all()
        out = Mat(ctx, shape=(rows, cols), pad=pad, off=off)
        _lib.call("orca_hip_act8_unpack", ctx.handle, p.ptr, rows, cols, _lib.F32, out.ptr, out.ld)
        np.testing.assert_array_equal(out.get(), value.astype(np.float32))
        half = ctx.upload(np.full(rows * (cols + pad) + 8, 0x1234, np.uint16))
        _lib.call("orca_hip_act8_unpack", ctx.handle, p.ptr, rows, cols, _lib.BF16, half.ptr + 2 * off, cols + pad)
        h = half.download(np.uint16, rows * (cols + pad) + 8)
        body = h[off:off + rows * (cols + pad)].reshape(rows, cols + pad)
        np.testing.assert_array_equal((body[:, :cols].astype(np.uint32) << 16).view(np.float32), value.astype(np.float32))
        assert (body[:, cols:] == 0x1234).all() and (h[:off] == 0x1234).all()


def test_pack_of_infinities_and_nan(ctx):
    x = np.ones((3, 70), np.float32)
    x[0, 3], x[1, 40], x[2, 69] = np.inf, np.nan, -np.inf
    p = Packed(ctx, 3, 70)
    X = Mat(ctx, x)
    _lib.call("orca_hip_act8_pack", ctx.handle, X.ptr, 3, 70, 70, p.ptr)
    assert p.get()[1].tolist() == [[255, 127, 127], [127, 255, 127], [127, 127, 255]]
    out = Mat(ctx, shape=(3, 70))
    _lib.call("orca_hip_act8_unpack", ctx.handle, p.ptr, 3, 70, _lib.F32, out.ptr, 70)
    got = out.get()
    bad = np.zeros((3, 70), bool)
    bad[0, :32] = bad[1, 32:64] = bad[2, 64:] = True
    np.testing.assert_array_equal(np.isnan(got), bad)
    assert (got[~bad] == 1.0).all()
    # as the input of a weight gradient: the groups' rows of dW, and no others, are NaN
    dw = Mat(ctx, shape=(70, 40))
    backward(ctx, Mat(ctx, np.ones((3, 40), np.float32)), Mat(ctx, np.zeros((70, 40), np.float32)), x8=p, dw=dw)
    got = dw.get()
    assert np.isnan(got).all()  # each group holds one of the three


def test_results_repeat_bit_for_bit(ctx):
    rng = np.random.default_rng(12)
    for m, n, k in [(4, 1000, 3001), (100, 300, 2000), (600, 520, 300)]:
        x, w, b, r = data(rng, m, n, k)
        X, W, B, R = Mat(ctx, x), Mat(ctx, w), Mat(ctx, b), Mat(ctx, r)
        first = None
        for _ in range(3):
            pre = Mat(ctx, shape=(m, n))
            dx, dw, db = Mat(ctx, shape=(m, k)), Mat(ctx, shape=(k, n)), Mat(ctx, shape=(1, n))
            y = forward(ctx, X, W, "gelu", B, R, pre).get()
            backward(ctx, R, W, "gelu", z=pre, x=X, dx=dx, dw=dw, db=db)
            got = [y, pre.get(), dx.get(), dw.get(), db.get()]
            first = first or got
            for a, c in zip(first, got):
                np.testing.assert_array_equal(a, c)


def test_one_row_equals_its_place_in_a_batch_to_rounding(ctx):
    rng = np.random.default_rng(13)
    m, n, k = 300, 260, 400
    x, w, b, r = data(rng, m, n, k)
    W, B = Mat(ctx, w), Mat(ctx, b)
    whole = forward(ctx, Mat(ctx, x), W, "silu", B, Mat(ctx, r)).get()
    s = np.abs(x).astype(np.float64) @ np.abs(w) + np.abs(b)
    for i in (0, 131, 299):
        one = forward(ctx, Mat(ctx, x[i:i + 1]), W, "silu", B, Mat(ctx, r[i:i + 1])).get()
        close(one, whole[i:i + 1].astype(np.float64), 2 * (act_tol(s[i:i + 1], product_tol(s[i:i + 1], k)) + 4 * U * 4),
              f"row {i}")
