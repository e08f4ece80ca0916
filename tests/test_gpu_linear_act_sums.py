"""Long sums of the fused Linear, with inputs that show what is left out: sums of zeros and ones that
grow with every row, and products of one term each at every place of a long k."""
from __future__ import annotations

import numpy as np
import pytest

from orcaml_amd import _lib
from orcaml_amd.device import Context
from tests import test_gpu_linear_act as L

pytestmark = pytest.mark.gpu


def flags(shape, odd, eighths):
    """A matrix of truth values, `eighths` / 8 of them true, spread evenly in another order for each odd multiplier."""
    h = np.arange(int(np.prod(shape)), dtype=np.uint32)
    h *= np.uint32(odd)
    return ((h >> np.uint32(29)) < eighths).reshape(shape)


def counts(a, b):
    """a [p][L], b [q][L] -> [p][q]: how often both are true."""
    if a.shape[1] < 1000:
        return a.astype(np.float32) @ b.T.astype(np.float32)
    b = [np.ascontiguousarray(r) for r in b]
    return np.array([[np.count_nonzero(r & c) for c in b] for r in map(np.ascontiguousarray, a)], np.float64)


@pytest.mark.parametrize("m,n,k", [(1, (1 << 25) + 5, 1), (3, 17000003, 2), ((1 << 25) + 5, 1, 1), (40000000, 2, 3),
                                   (20, 17000001, 1), (1, 2, 17000001)])
def test_the_longest_sums_count_every_term(ctx, m, n, k):
    """Zeros and ones: every partial sum is a whole number below 2^24, in any order exact, and a row, a column or a
    split that is left out, taken twice or taken from elsewhere is missing in the count."""
    x, w = flags((m, k), 2654435761, 7), flags((k, n), 2246822519, 4)
    dy, z = flags((m, n), 3266489917, 4), flags((m, n), 668265263, 6)
    g = dy & z
    want = {"y": counts(x, w.T), "dx": counts(g, w), "dw": counts(x.T, g.T), "db": np.count_nonzero(g, 0)[None]}
    for what, v in want.items():
        assert v.max() < 1 << 24, what
    X, W, DY = (L.Mat(ctx, v.astype(np.float32)) for v in (x, w, dy))
    Z = L.Mat(ctx, np.where(z, np.float32(1), np.float32(-1)))
    x8, z8 = L.Packed(ctx, m, k), L.Packed(ctx, m, n)  # exact: 64 steps of 2^-6, or zeros
    for of, p in ((X, x8), (Z, z8)):
        _lib.call("orca_hip_act8_pack", ctx.handle, of.ptr, of.rows, of.cols, of.ld, p.ptr)
    np.testing.assert_array_equal(L.forward(ctx, X, W).get(), want["y"])
    for kept, saved in (("fp32", dict(x=X, z=Z)), ("8bit", dict(x8=x8, z8=z8))):
        print(f"longest {m}x{n}x{k} {kept}", flush=True)
        out = {"dx": L.Mat(ctx, shape=(m, k)), "dw": L.Mat(ctx, shape=(k, n)), "db": L.Mat(ctx, shape=(1, n))}
        L.backward(ctx, DY, W, "relu", **saved, **out)
        for what, t in out.items():
            np.testing.assert_array_equal(t.get(), want[what], err_msg=f"{what} {kept}")


@pytest.fixture(scope="module", params=[(64, 1), (64, 12), (128, 1), (128, 5), (256, 1), (256, 4), (0, 0)],
                ids=lambda p: f"tile{p[0]}-splits{p[1]}")
def tiled(request):
    with pytest.MonkeyPatch.context() as mp:
        if request.param[0]:
            mp.setenv("ORCA_HIP_LINEAR_TILE", str(request.param[0]))
            mp.setenv("ORCA_HIP_LINEAR_SPLITS", str(request.param[1]))
        c = Context(0)
    yield c
    c.close()


def full(rng, shape):
    """Values of 24 significant bits each."""
    v = rng.integers(1 << 23, 1 << 24, shape) | 1
    return (v * rng.choice([-1.0, 1.0], shape) * 2.0 ** -23).astype(np.float32)


def scattered(rng, rows, cols):
    """One value of 24 bits in every column, its rows spread from the first to the last."""
    v = np.zeros((rows, cols), np.float32)
    at = rng.integers(0, rows, cols)
    at[:4] = 0, rows - 1, rows // 2, rows - 2
    v[at, np.arange(cols)] = full(rng, cols)
    return v


@pytest.mark.parametrize("long", [4100, 9001])
def test_every_term_of_a_long_product(tiled, long):
    """A sum of one product x w, and of zeros.  With x = h + m + l, |m| <= 2^-7 |x| and |l| <= 2^-16 |x|: the three terms
    left out are at most 2^-23, 2^-23 and 2^-32 of x w, and six terms are added, each addition off by at most 2^-23 (however
    the instruction rounds): less than 2^-20 of x w in all.  Any of the six left out is up to 2^-14 of it, and a k left out
    all of it."""
    rng = np.random.default_rng(long)
    a, b = 270, 300
    tol = 2.0 ** -20

    def check(got, want, what):
        L.close(got, want, tol * np.abs(want), what)

    f64 = np.float64
    x, w = full(rng, (a, long)), scattered(rng, long, b)
    check(L.forward(tiled, L.Mat(tiled, x), L.Mat(tiled, w)).get(), x.astype(f64) @ w.astype(f64), "y")
    w2 = scattered(rng, long, b).T.copy()  # [b][long]: dx sums over its columns
    dx = L.Mat(tiled, shape=(a, b))
    L.backward(tiled, L.Mat(tiled, x), L.Mat(tiled, w2), dx=dx)
    check(dx.get(), x.astype(f64) @ w2.T.astype(f64), "dx")
    x3, dy = full(rng, (long, a)), scattered(rng, long, b)
    dw = L.Mat(tiled, shape=(a, b))
    L.backward(tiled, L.Mat(tiled, dy), L.Mat(tiled, shape=(a, b)), x=L.Mat(tiled, x3), dw=dw)
    check(dw.get(), x3.T.astype(f64) @ dy.astype(f64), "dw")
    # from a checkpoint: its values are one term, so nothing is left out but roundings of three
    codes, steps = rng.integers(1, 128, (long, a)) * rng.choice([-1, 1], (long, a)), rng.integers(120, 135, (long, -(-a // 32)))
    L.backward(tiled, L.Mat(tiled, dy), L.Mat(tiled, shape=(a, b)), x8=L.Packed(tiled, long, a, L.write_packed(codes, steps)),
               dw=dw)
    check(dw.get(), L.value64(codes, steps).T @ dy.astype(f64), "dw from a checkpoint")


@pytest.mark.parametrize("m,n,k,takes", [(1100, 4099, 2051, "linear_act_t256"),
                                         (2100, 2051, 2051, "linear_act_backward_t256")])
def test_layers_that_take_the_largest_tile(ctx, m, n, k, takes):
    """The cost model's own choice of the 256 tile, on whole numbers: exact."""
    rng = np.random.default_rng(3)

    def whole(shape, top):
        return rng.integers(-top, top + 1, shape).astype(np.float32)

    x, w, dy = whole((m, k), 40), whole((k, n), 6), whole((m, n), 6)
    X, W, DY = L.Mat(ctx, x), L.Mat(ctx, w), L.Mat(ctx, dy)
    dx, dw, db = L.Mat(ctx, shape=(m, k)), L.Mat(ctx, shape=(k, n)), L.Mat(ctx, shape=(1, n))
    ctx.prof_reset()
    ctx.prof_enable(True)
    y = L.forward(ctx, X, W)
    L.backward(ctx, DY, W, x=X, dx=dx, dw=dw, db=db)
    ctx.prof_enable(False)
    names = [q["name"].split()[0] for q in ctx.prof_report()["kernels"]]
    assert takes in names, names
    # sums below 2^24 of whole numbers, so exact in fp32 too
    np.testing.assert_array_equal(y.get(), x @ w)
    np.testing.assert_array_equal(dx.get(), dy @ w.T)
    np.testing.assert_array_equal(dw.get(), x.T @ dy)
    np.testing.assert_array_equal(db.get(), dy.sum(0, keepdims=True))
