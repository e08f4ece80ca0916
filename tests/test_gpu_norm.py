"""orca_hip_norm, orca_hip_residual_norm, their backward passes and orca_hip_dropout against the formulas in 64
bits (tests/norm_oracle.py derives the tolerances): kinds of norm, gates and lengths, odd sizes, strides, what lies
between the rows, calls in place, rows of NaN, repeated calls."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from orcaml_amd import _lib
from tests import norm_oracle as O
from tests.norm_oracle import U
from tests.test_gpu_linear_act import layout, pack64, read_packed

pytestmark = pytest.mark.gpu

NORMS = ["none", "layer", "rms"]
EPS = 1e-5


class Matrix:
    """A matrix [rows][cols] in device memory with a leading dimension and a start that need not be aligned, and known
    values before, between and behind its rows."""

    GAP = -7.25

    def __init__(self, ctx, rows, cols, values=None, ld=None, start=0):
        self.rows, self.cols, self.ld, self.start = rows, cols, ld or cols, start
        self.host = np.full(start + max(rows, 1) * self.ld + 5, self.GAP, np.float32)
        if values is not None:
            self.view(self.host)[:] = values
        self.buf = ctx.upload(self.host)
        self.ptr = self.buf.ptr + 4 * start

    def view(self, flat):
        return flat[self.start:self.start + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    def read(self):
        """Its values; what lies around them must be untouched."""
        flat = self.buf.download(count=self.host.size)
        got = self.view(flat).copy()
        self.view(flat)[:] = self.GAP
        assert (flat == self.GAP).all(), "values around the matrix were written"
        return got


def params(kind, w, b, eps=EPS):
    return _lib.NormParams(kind=NORMS.index(kind), eps=eps, weight=w.ptr if w else None, bias=b.ptr if b else None)


def close(got, want, what):
    value, tol = want
    err = np.abs(got.astype(np.float64) - value)
    bad = ~(err <= tol + 1e-42)
    assert not bad.any(), (what, int(bad.sum()), float((err / (tol + 1e-42)).max()), np.argwhere(bad)[:3].tolist())


def stream(rng, m, n, mean=0.5):
    return ((rng.standard_normal((m, n)) + mean) * np.exp(0.5 * rng.standard_normal((1, n)))).astype(np.float32)


class Joint:
    """Inputs of a joint, in 64 bits for the oracle and on the device for the call."""

    def __init__(self, ctx, seed, m, n, post="none", next="none", groups=0, p=0.0, bias=True, weight=True, rs=1.0,
                 bs=1.0, pad=0, start=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.m, self.n, self.pad, self.start = ctx, m, n, pad, start
        self.seed, self.offset, self.p, self.groups = seed * 0x9E3779B97F4A7C15 % 2 ** 64, seed * 977 + (5 << 40), p, groups
        self.host = {"x": stream(rng, m, n), "f": stream(rng, m, n), "dy": stream(rng, m, n, 0.0),
                     "du": stream(rng, m, n, 0.0)}
        vec = {}
        for name, kind in (("post", post), ("next", next)):
            if kind == "none":
                continue
            if weight:
                vec[name + "_w"] = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32)
            if bias:
                vec[name + "_b"] = (0.3 * rng.standard_normal(n)).astype(np.float32)
        self.gate = (0.7 + 0.4 * rng.standard_normal((groups, n))).astype(np.float32) if groups else None
        self.dev = {k: self.matrix(v) for k, v in self.host.items()}
        self.vec = {k: ctx.upload(v) for k, v in vec.items()}
        self.dgate_in = self.matrix(self.gate) if groups else None

        def spec(name, kind):
            return (kind, EPS, vec.get(name + "_w", np.ones(n)).astype(np.float64),
                    vec.get(name + "_b", np.zeros(n)).astype(np.float64))

        self.oracle = {"post": spec("post", post), "next": spec("next", next),
                       "gate": None if self.gate is None else self.gate.astype(np.float64),
                       "rs": float(np.float32(rs)), "bs": float(np.float32(bs)),
                       "factor": O.dropout_factor(m, n, p, self.seed, self.offset)}
        self.block = _lib.ResidualBlock(
            post=params(post, self.vec.get("post_w"), self.vec.get("post_b")),
            next=params(next, self.vec.get("next_w"), self.vec.get("next_b")),
            gate=self.dgate_in.ptr if groups else None, groups=groups, ldgate=self.dgate_in.ld if groups else 0,
            residual_scale=rs, block_scale=bs, p=p, seed=self.seed, offset=self.offset)
        self.post, self.next = post, next

    def matrix(self, values=None, rows=None):
        rows = values.shape[0] if values is not None else rows if rows is not None else self.m
        return Matrix(self.ctx, rows, self.n, values, self.n + self.pad, self.start)

    def forward(self, packed=False):
        d, y = self.dev, self.matrix()
        u = self.matrix() if self.next != "none" else None
        u8 = self.ctx.alloc(layout(self.m, self.n)[3]) if packed else None
        _lib.call("orca_hip_residual_norm", self.ctx.handle, self.m, self.n, d["x"].ptr, d["x"].ld, d["f"].ptr,
                  d["f"].ld, ctypes.byref(self.block), y.ptr, y.ld, u.ptr if u else None, u.ld if u else 0,
                  u8.ptr if packed else None)
        out = {"y": y.read()}
        if u:
            out["u"] = u.read()
        if packed:
            out["u8"] = u8.download(np.uint8)
        return out

    def backward(self, y, dy=True, du=True, want=None, dx_over_dy=False):
        du = du and self.next != "none"
        d, ym = self.dev, self.matrix(y)
        names = ["dx", "df"] + (["dgate"] if self.groups else [])
        names += ["dpost_weight", "dpost_bias"] if self.post != "none" else []
        names += ["dnext_weight", "dnext_bias"] if du else []
        names = [k for k in names if want is None or k in want]
        out = {k: self.matrix(rows={"dx": self.m, "df": self.m, "dgate": self.groups}.get(k, 1)) for k in names}
        if dx_over_dy:
            out["dx"] = self.matrix(self.host["dy"])
        g = _lib.ResidualGrads(**{k: v.ptr for k, v in out.items()})
        g.lddx = g.lddf = g.lddgate = self.n + self.pad
        dyp = out["dx"] if dx_over_dy else d["dy"]
        _lib.call("orca_hip_residual_norm_backward", self.ctx.handle, self.m, self.n, dyp.ptr if dy else None, dyp.ld,
                  d["du"].ptr if du else None, d["du"].ld, d["f"].ptr, d["f"].ld, ym.ptr, ym.ld,
                  ctypes.byref(self.block), ctypes.byref(g))
        return {k: v.read() for k, v in out.items()}

    def want_forward(self):
        return O.joint(self.host["x"].astype(np.float64), self.host["f"].astype(np.float64), self.oracle)

    def want_backward(self, y, dy=True, du=True):
        h = {k: v.astype(np.float64) for k, v in self.host.items()}
        return O.joint_back(h["dy"] if dy else None, h["du"] if du and self.next != "none" else None, h["f"],
                            y.astype(np.float64), self.oracle)

    def check(self):
        got, want = self.forward(), self.want_forward()
        assert set(got) == set(want)
        for k in got:
            close(got[k], want[k], k)
        back, wb = self.backward(got["y"]), self.want_backward(got["y"])
        for k, v in back.items():
            value, tol = wb[k]
            close(v, (value.reshape(v.shape), tol.reshape(v.shape)), k)
        return got, back


# lengths around every edge of a kernel: a quad, a wave's quads, rows in registers, rows in passes
LENGTHS = [1, 2, 3, 4, 5, 7, 8, 31, 33, 64, 100, 255, 256, 257, 511, 512, 516, 1000, 1003, 1023, 1024, 1025, 1501, 2044, 2048,
           2049, 3001, 4095, 4096, 4097, 6001, 8191, 8192, 8193, 16384, 16385, 20001]


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("pad,start", [(0, 0), (3, 1)])
def test_norm(ctx, n, kind, pad, start):
    m = 5 if n < 4000 else 3
    print(f"norm {m} x {n} {kind} pad {pad}", flush=True)
    rng = np.random.default_rng(n)
    x, dy, add = stream(rng, m, n), stream(rng, m, n, 0.0), stream(rng, m, n, 0.0)
    w, b = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    mx, mdy, madd, my, mdx = (Matrix(ctx, m, n, v, n + pad, start) for v in (x, dy, add, None, None))
    dw, db = Matrix(ctx, 1, n, start=start), Matrix(ctx, 1, n, start=start)
    p = params(kind, ctx.upload(w), ctx.upload(b))
    wb = ctx.upload(w), ctx.upload(b)
    p.weight, p.bias = wb[0].ptr, wb[1].ptr
    _lib.call("orca_hip_norm", ctx.handle, m, n, mx.ptr, mx.ld, ctypes.byref(p), my.ptr, my.ld, None)
    x64, w64, b64 = x.astype(np.float64), w.astype(np.float64), b.astype(np.float64)
    close(my.read(), O.norm(kind, x64, EPS, w64, b64), "y")
    _lib.call("orca_hip_norm_backward", ctx.handle, m, n, mdy.ptr, mdy.ld, mx.ptr, mx.ld, ctypes.byref(p), madd.ptr,
              madd.ld, mdx.ptr, mdx.ld, dw.ptr, db.ptr)
    (d, td), (vw, tw), (vb, tb) = O.norm_back(kind, x64, EPS, w64, dy.astype(np.float64))
    total = d + add
    close(mdx.read(), (total, td + 2 * U * (np.abs(d) + np.abs(add))), "dx")
    close(dw.read(), (vw[None], tw[None]), "dw")
    close(db.read(), (vb[None], tb[None]), "db")


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 17, 63, 64, 65, 255, 300, 1030])
@pytest.mark.parametrize("n", [8, 64, 130, 1024])
def test_norm_sums_over_rows(ctx, m, n):
    print(f"norm rows {m} x {n}", flush=True)
    rng = np.random.default_rng(m * n)
    x, dy = stream(rng, m, n), stream(rng, m, n, 0.2)
    mx, mdy, dw, db = (Matrix(ctx, r, n, v) for r, v in ((m, x), (m, dy), (1, None), (1, None)))
    p = params("layer", None, None)
    _lib.call("orca_hip_norm_backward", ctx.handle, m, n, mdy.ptr, n, mx.ptr, n, ctypes.byref(p), None, 0, None, 0,
              dw.ptr, db.ptr)
    _, (vw, tw), (vb, tb) = O.norm_back("layer", x.astype(np.float64), EPS, np.ones(n), dy.astype(np.float64))
    close(dw.read(), (vw[None], tw[None]), "dw")
    close(db.read(), (vb[None], tb[None]), "db")


@pytest.mark.parametrize("post", NORMS)
@pytest.mark.parametrize("next", NORMS)
@pytest.mark.parametrize("groups", [0, 1, 4, 12])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_joint_parts(ctx, post, next, groups, p):
    print(f"joint {post} {next} groups {groups} p {p}", flush=True)
    for n in (36, 1003):
        Joint(ctx, n + groups, 12, n, post, next, groups, p, rs=0.75, bs=1.5).check()


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("pad,start", [(0, 0), (3, 1)])
def test_joint_lengths(ctx, n, pad, start):
    print(f"joint 6 x {n} pad {pad}", flush=True)
    Joint(ctx, n, 6, n, "layer", "rms", 3, 0.2, pad=pad, start=start).check()
    Joint(ctx, n, 2, n, "rms", "layer", 2, 0.0, pad=pad, start=start).check()


# one group of many rows, many groups of few, groups that one block sums and groups that several do
@pytest.mark.parametrize("m,groups", [(1, 1), (2, 1), (70, 1), (70, 2), (70, 35), (70, 70), (600, 3), (600, 200), (1200, 600),
                                      (2100, 2100), (4200, 1400), (3000, 2)])
@pytest.mark.parametrize("n", [24, 260])
def test_joint_gates(ctx, m, groups, n):
    print(f"joint gates {m} x {n} groups {groups}", flush=True)
    Joint(ctx, m + groups, m, n, "rms", "layer", groups, 0.1).check()
    Joint(ctx, m + groups, m, n, "none", "none", groups, 0.0).check()


# more rows than the blocks take at once, in each length of row that has kernels of its own
@pytest.mark.parametrize("m,n", [(3000, 256), (9000, 50), (2500, 400), (5000, 700), (1000, 1500), (2000, 4096), (1100, 2600),
                                 (700, 6000)])
@pytest.mark.parametrize("bias", [False, True])
def test_joint_large(ctx, m, n, bias):
    print(f"joint large {m} x {n} bias {bias}", flush=True)
    Joint(ctx, m, m, n, "rms", "rms", 1, 0.1, bias=bias).check()
    if bias:
        Joint(ctx, m + 1, m, n, "none", "layer", 0, 0.0, bias=bias).check()


# each kernel: the lengths of a row that have one, the norms that are there, with biases and without
@pytest.mark.parametrize("n", [200, 401, 1000, 1502, 3003, 6000])
@pytest.mark.parametrize("post", NORMS)
@pytest.mark.parametrize("next", NORMS)
@pytest.mark.parametrize("bias", [False, True])
def test_every_kernel(ctx, n, post, next, bias):
    print(f"kernels {n} {post} {next} {bias}", flush=True)
    for groups, p in ((0, 0.1), (1, 0.0), (3, 0.0), (9, 0.3)):
        Joint(ctx, n + groups, 9, n, post, next, groups, p, bias=bias).check()


def test_without_weights(ctx):
    for n in (100, 1030):
        Joint(ctx, n, 9, n, "layer", "rms", 0, 0.1, bias=False, weight=False).check()


def test_gradients_of_one_side(ctx):
    """dy or du alone, and any part of the results alone, with the same bits."""
    for n in (52, 900, 1500, 4000, 8200):
        j = Joint(ctx, n, 40, n, "layer", "layer", 4, 0.25, rs=0.5)
        y = j.forward()["y"]
        full = j.backward(y)
        for k in full:
            np.testing.assert_array_equal(j.backward(y, want={k})[k], full[k], err_msg=k)
        for sides in ({"dy": False}, {"du": False}):
            got, want = j.backward(y, **sides), j.want_backward(y, **sides)
            for k, v in got.items():
                close(v, tuple(t.reshape(v.shape) for t in want[k]), (k, sides))
        np.testing.assert_array_equal(j.backward(y, dx_over_dy=True)["dx"], full["dx"])


def test_same_bits_every_time(ctx):
    j = Joint(ctx, 3, 2500, 300, "rms", "layer", 5, 0.1)
    a, b = j.forward(), j.forward()
    for k in a:
        np.testing.assert_array_equal(a[k], b[k])
    one, two = j.backward(a["y"]), j.backward(a["y"])
    for k in one:
        np.testing.assert_array_equal(one[k], two[k])


def test_in_place(ctx):
    for n in (40, 1003, 9000):
        rng = np.random.default_rng(n)
        x = stream(rng, 7, n)
        apart, over = Matrix(ctx, 7, n), Matrix(ctx, 7, n, x)
        src, p = Matrix(ctx, 7, n, x), params("layer", None, None)
        _lib.call("orca_hip_norm", ctx.handle, 7, n, src.ptr, n, ctypes.byref(p), apart.ptr, n, None)
        _lib.call("orca_hip_norm", ctx.handle, 7, n, over.ptr, n, ctypes.byref(p), over.ptr, n, None)
        np.testing.assert_array_equal(over.read(), apart.read())
        j = Joint(ctx, n, 7, n, "rms", "layer", 7, 0.1)
        want = j.forward()
        x, u = j.matrix(j.host["x"]), j.matrix()
        _lib.call("orca_hip_residual_norm", ctx.handle, 7, n, x.ptr, n, j.dev["f"].ptr, n, ctypes.byref(j.block), x.ptr,
                  n, u.ptr, n, None)
        np.testing.assert_array_equal(x.read(), want["y"])
        np.testing.assert_array_equal(u.read(), want["u"])
        dy, add = j.dev["dy"], j.matrix(j.host["du"])
        outs = []
        for into in (j.matrix(), add):
            _lib.call("orca_hip_norm_backward", ctx.handle, 7, n, dy.ptr, n, j.dev["f"].ptr, n, ctypes.byref(p),
                      add.ptr, n, into.ptr, n, None, None)
            outs.append(into.read())
        np.testing.assert_array_equal(outs[0], outs[1])


@pytest.mark.parametrize("m,n", [(3, 1), (4, 3), (5, 8), (17, 33), (40, 1003), (16, 1024), (3, 4100), (2, 9001)])
def test_checkpoint_of_the_output(ctx, m, n):
    """The checkpoint is that of the values written, and writing it changes none of them."""
    rng = np.random.default_rng(n)
    x, p = Matrix(ctx, m, n, stream(rng, m, n)), params("layer", None, None)
    y, y8 = Matrix(ctx, m, n), ctx.alloc(layout(m, n)[3])
    plain = Matrix(ctx, m, n)
    _lib.call("orca_hip_norm", ctx.handle, m, n, x.ptr, n, ctypes.byref(p), y.ptr, n, y8.ptr)
    _lib.call("orca_hip_norm", ctx.handle, m, n, x.ptr, n, ctypes.byref(p), plain.ptr, n, None)
    np.testing.assert_array_equal(y.read(), plain.read())
    codes, bytes_ = pack64(y.read())
    got_codes, got_bytes = read_packed(y8.download(np.uint8), m, n)
    np.testing.assert_array_equal(got_bytes, bytes_)
    np.testing.assert_array_equal(got_codes, codes)
    j = Joint(ctx, n, m, n, "none", "rms", 0, 0.2, pad=2, start=3)
    out = j.forward(packed=True)
    np.testing.assert_array_equal(out["u"], j.forward()["u"])
    codes, bytes_ = pack64(out["u"])
    got_codes, got_bytes = read_packed(out["u8"], m, n)
    np.testing.assert_array_equal(got_bytes, bytes_)
    np.testing.assert_array_equal(got_codes, codes)


@pytest.mark.parametrize("n", [12, 700, 3000, 9000])
def test_bad_rows_keep_to_themselves(ctx, n):
    """NaN and infinities in a row change no other row; dropped values are 0 whatever they were."""
    j = Joint(ctx, n, 9, n, "none", "layer", 9, 0.5)
    clean = j.forward()
    clean_back = j.backward(clean["y"])
    f = j.host["f"].copy()
    f[2, 5], f[6, n - 1], f[7] = np.nan, np.inf, -np.inf
    j.dev["f"] = j.matrix(f)
    got = j.forward()
    rows = [r for r in range(9) if r not in (2, 6, 7)]
    np.testing.assert_array_equal(got["y"][rows], clean["y"][rows])
    np.testing.assert_array_equal(got["u"][rows], clean["u"][rows])
    dropped = j.oracle["factor"] == 0
    np.testing.assert_array_equal(got["y"][dropped], j.host["x"][dropped])
    back = j.backward(clean["y"])
    np.testing.assert_array_equal(back["df"], clean_back["df"])  # without a post norm f is no part of it
    np.testing.assert_array_equal(back["dgate"][rows], clean_back["dgate"][rows])
    assert (back["dgate"][dropped] == 0).all()


@pytest.mark.parametrize("n", [7, 300, 1000, 2000, 4000, 8000, 9000])
def test_what_a_bad_value_makes_of_its_row(ctx, n):
    """As the formulas in fp32: NaN throughout, but 0 at the finite values of an rms row with an infinity."""
    rng = np.random.default_rng(n)
    x, w, b = stream(rng, 6, n), (1 + rng.random(n)).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    x[1, 3], x[3, n - 1], x[4, 0] = np.nan, np.inf, -np.inf
    mx, my, dy, dx = Matrix(ctx, 6, n, x), Matrix(ctx, 6, n), Matrix(ctx, 6, n, stream(rng, 6, n)), Matrix(ctx, 6, n)
    ws = ctx.upload(w), ctx.upload(b)
    for kind in ("layer", "rms"):
        p = params(kind, *ws)
        _lib.call("orca_hip_norm", ctx.handle, 6, n, mx.ptr, n, ctypes.byref(p), my.ptr, n, None)
        got = my.read()
        assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2, 5]]).all()
        for row, col in ((3, n - 1), (4, 0)):
            rest = np.arange(n) != col
            assert np.isnan(got[row, col])
            if kind == "layer":
                assert np.isnan(got[row]).all()
            else:
                np.testing.assert_array_equal(got[row][rest], b[rest])
        _lib.call("orca_hip_norm_backward", ctx.handle, 6, n, dy.ptr, n, mx.ptr, n, ctypes.byref(p), None, 0, dx.ptr, n,
                  None, None)
        got = dx.read()
        assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2, 5]]).all()


def test_rows_of_one_value(ctx):
    """A row of equal values has no deviation: layer gives the bias, whatever the value; rms of zeros as well."""
    for n in (5, 100, 1000, 4097, 12000):
        b = np.random.default_rng(n).standard_normal(n).astype(np.float32)
        bias = ctx.upload(b)
        x, y = Matrix(ctx, 4, n, np.repeat(np.float32([[0.1], [1000.7], [-3e5], [0.0]]), n, 1)), Matrix(ctx, 4, n)
        for kind in ("layer", "rms"):
            _lib.call("orca_hip_norm", ctx.handle, 4, n, x.ptr, n, ctypes.byref(params(kind, None, bias)), y.ptr, n, None)
            got = y.read()
            np.testing.assert_array_equal(got[3], b)
            if kind == "layer":
                # the sum of the differences corrects the mean to (steps + 2) U of the first mean's error, steps U |v|
                v = np.abs(np.float64([[0.1], [1000.7], [-3e5], [0.0]]))
                assert (np.abs(got - b) <= (O.steps(n) + 2) ** 2 * U ** 2 * v / np.sqrt(EPS) + 2 * U * np.abs(b)).all()


def test_a_large_common_part(ctx):
    """A mean of 1000 deviations costs the digits that fp32 inputs lose, and no more."""
    for n in (64, 1000, 4096, 10000):
        rng = np.random.default_rng(n)
        x = (rng.standard_normal((6, n)) + 1000).astype(np.float32)
        mx, my = Matrix(ctx, 6, n, x), Matrix(ctx, 6, n)
        _lib.call("orca_hip_norm", ctx.handle, 6, n, mx.ptr, n, ctypes.byref(params("layer", None, None)), my.ptr, n, None)
        close(my.read(), O.norm("layer", x.astype(np.float64), EPS, np.ones(n), np.zeros(n)), n)


@pytest.mark.parametrize("n", [1, 3, 4, 5, 40, 255, 256, 257, 784, 1003, 4100])
@pytest.mark.parametrize("m", [1, 3, 17, 70])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(ctx, m, n, p):
    print(f"dropout {m} x {n} p {p}", flush=True)
    rng = np.random.default_rng(m + n)
    x = rng.standard_normal((m, n)).astype(np.float32)
    x[0, 0] = np.inf
    seed, offset = 0x0123456789ABCDEF * (n + 1) % 2 ** 64, (n << 33) + m
    factor = O.dropout_factor(m, n, p, seed, offset)
    for pad, start in ((0, 0), (3, 2)):
        mx, my = Matrix(ctx, m, n, x, n + pad, start), Matrix(ctx, m, n, None, n + pad, start)
        _lib.call("orca_hip_dropout", ctx.handle, m, n, mx.ptr, mx.ld, p, seed, offset, my.ptr, my.ld)
        got = my.read()
        kept = factor > 0
        np.testing.assert_array_equal(got[~kept], 0.0)
        want = x[kept].astype(np.float64) * factor[kept]
        # the scale and the product are rounded once each
        with np.errstate(invalid="ignore"):  # the infinity
            assert ((np.abs(got[kept] - want) <= 3 * U * np.abs(want)) | (got[kept] == want)).all()
        _lib.call("orca_hip_dropout", ctx.handle, m, n, mx.ptr, mx.ld, p, seed, offset, mx.ptr, mx.ld)
        np.testing.assert_array_equal(mx.read(), got)


def test_dropout_draws_apart(ctx):
    """Other seeds and offsets draw other masks: two masks of 4096 fair values agree in 2048 +- 6 * 32 places."""
    x, y = Matrix(ctx, 8, 512, np.ones((8, 512), np.float32)), Matrix(ctx, 8, 512)
    masks = []
    for seed, offset in ((0, 0), (1, 0), (0, 1), (1 << 32, 0), (0, 1 << 32)):
        _lib.call("orca_hip_dropout", ctx.handle, 8, 512, x.ptr, 512, 0.5, seed, offset, y.ptr, 512)
        masks.append(y.read() > 0)
    for i in range(5):
        for k in range(i):
            assert abs(int((masks[i] == masks[k]).sum()) - 2048) < 192


def test_nothing_to_do(ctx):
    """Sizes of zero: nothing is written but the sums of no rows."""
    p = params("rms", None, None)
    one = Matrix(ctx, 1, 8)
    for m, n in ((0, 8), (8, 0), (0, 0)):
        _lib.call("orca_hip_norm", ctx.handle, m, n, None, n, ctypes.byref(p), None, n, None)
        _lib.call("orca_hip_dropout", ctx.handle, m, n, None, n, 0.5, 1, 2, None, n)
        b = _lib.ResidualBlock(next=p, residual_scale=1.0, block_scale=1.0)
        _lib.call("orca_hip_residual_norm", ctx.handle, m, n, None, n, None, n, ctypes.byref(b), None, n, None, n, None)
    for gate_rows in (1, 3):
        dgate, dw, db = Matrix(ctx, gate_rows, 8, None, 11), Matrix(ctx, 1, 8), Matrix(ctx, 1, 8)
        gate = Matrix(ctx, gate_rows, 8, np.ones((gate_rows, 8), np.float32))
        b = _lib.ResidualBlock(post=p, next=p, gate=gate.ptr, groups=gate_rows, ldgate=8, residual_scale=1.0, block_scale=1.0)
        g = _lib.ResidualGrads(dgate=dgate.ptr, lddgate=11, dpost_weight=dw.ptr, dnext_bias=db.ptr)
        _lib.call("orca_hip_residual_norm_backward", ctx.handle, 0, 8, None, 8, one.ptr, 8, None, 8, None, 8, ctypes.byref(b),
                  ctypes.byref(g))
        for t in (dgate, dw, db):
            assert (t.read() == 0).all()


def test_operands_that_are_too_small_or_freed(ctx):
    """Found on the host, before any launch (blocks are whole multiples of 256 bytes)."""
    small, big, p = ctx.alloc(256), ctx.alloc(512), params("rms", None, None)
    with pytest.raises(_lib.OrcaHipError, match=r"norm \(x\)"):
        _lib.call("orca_hip_norm", ctx.handle, 8, 16, small.ptr, 16, ctypes.byref(p), big.ptr, 16, None)
    with pytest.raises(_lib.OrcaHipError, match=r"norm \(y\)"):
        _lib.call("orca_hip_norm", ctx.handle, 8, 16, big.ptr, 16, ctypes.byref(p), small.ptr, 16, None)
    with pytest.raises(_lib.OrcaHipError, match=r"dropout \(y\)"):
        _lib.call("orca_hip_dropout", ctx.handle, 8, 16, big.ptr, 16, 0.5, 0, 0, small.ptr, 16)
    b = _lib.ResidualBlock(next=p, gate=small.ptr, groups=8, ldgate=16, residual_scale=1.0, block_scale=1.0)
    others = [ctx.alloc(512) for _ in range(4)]
    with pytest.raises(_lib.OrcaHipError, match=r"residual_norm \(gate\)"):
        _lib.call("orca_hip_residual_norm", ctx.handle, 8, 16, big.ptr, 16, others[0].ptr, 16, ctypes.byref(b),
                  others[1].ptr, 16, others[2].ptr, 16, None)
    ptr = others.pop().ptr
    ctx.release_dropped()
    with pytest.raises(_lib.OrcaHipError, match="freed"):
        _lib.call("orca_hip_norm", ctx.handle, 8, 16, ptr, 16, ctypes.byref(p), big.ptr, 16, None)


def test_on_the_side_stream(ctx):
    """A forward runs there; a backward that needs a workspace is refused, and one block's, which needs none, runs."""
    j = Joint(ctx, 11, 600, 300, "rms", "layer", 1, 0.2)
    one = Joint(ctx, 12, 6, 300, "rms", "layer", 1, 0.2)
    want, want_one = j.forward(), one.backward(one.host["x"])
    d, y, u, dw = j.dev, j.matrix(), j.matrix(), j.matrix(rows=1)
    od, ody, odx = one.dev, one.matrix(one.host["x"]), one.matrix()
    ctx.sync()
    ctx.use_side_stream(-1)
    try:
        _lib.call("orca_hip_residual_norm", ctx.handle, j.m, j.n, d["x"].ptr, j.n, d["f"].ptr, j.n, ctypes.byref(j.block),
                  y.ptr, j.n, u.ptr, j.n, None)
        g = _lib.ResidualGrads(dx=odx.ptr, lddx=one.n)
        _lib.call("orca_hip_residual_norm_backward", ctx.handle, one.m, one.n, od["dy"].ptr, one.n, od["du"].ptr, one.n,
                  od["f"].ptr, one.n, ody.ptr, one.n, ctypes.byref(one.block), ctypes.byref(g))
        with pytest.raises(_lib.OrcaHipError, match="side stream"):
            _lib.call("orca_hip_norm_backward", ctx.handle, j.m, j.n, d["dy"].ptr, j.n, d["x"].ptr, j.n,
                      ctypes.byref(j.block.next), None, 0, None, 0, dw.ptr, None)
    finally:
        ctx.use_side_stream(0)
    ctx.sync()
    for k, m in (("y", y), ("u", u)):
        np.testing.assert_array_equal(m.read(), want[k])
    np.testing.assert_array_equal(odx.read(), want_one["dx"])


def test_another_context_on_its_own_stream(ctx):
    """Two contexts, so two streams, at once: each gives what it gives alone."""
    from orcaml_amd.device import Context

    other = Context(ctx.device)
    try:
        jobs = [Joint(c, s, 900, 520, "rms", "layer", 3, 0.1) for s, c in ((1, ctx), (2, other), (3, ctx), (4, other))]
        alone = [(j.forward(), j.backward(j.host["x"])) for j in jobs]
        bufs = []
        for j in jobs:  # enqueued on both streams with no wait between
            d, y, u = j.dev, j.matrix(), j.matrix()
            _lib.call("orca_hip_residual_norm", j.ctx.handle, j.m, j.n, d["x"].ptr, j.n, d["f"].ptr, j.n,
                      ctypes.byref(j.block), y.ptr, j.n, u.ptr, j.n, None)
            dx, df, dw = j.matrix(), j.matrix(), j.matrix(rows=1)
            g = _lib.ResidualGrads(dx=dx.ptr, lddx=j.n, df=df.ptr, lddf=j.n, dnext_weight=dw.ptr)
            _lib.call("orca_hip_residual_norm_backward", j.ctx.handle, j.m, j.n, d["dy"].ptr, j.n, d["du"].ptr, j.n,
                      d["f"].ptr, j.n, d["x"].ptr, j.n, ctypes.byref(j.block), ctypes.byref(g))
            bufs.append({"y": y, "u": u, "dx": dx, "df": df, "dnext_weight": dw})
        for (fwd, back), b in zip(alone, bufs):
            for k, v in b.items():
                np.testing.assert_array_equal(v.read(), {**fwd, **back}[k])
        del jobs, bufs
    finally:
        other.close()
