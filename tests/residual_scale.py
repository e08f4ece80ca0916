"""The gradients of a joint's output and of its stream at any residual scale, on the CPU and on the GPU."""
from __future__ import annotations

import numpy as np

from orcaml_amd import autodiff as A
from tests.norm_oracle import U

# the ends of the range that a joint takes, scales whose products with a gradient leave fp32's range, ordinary ones
SCALES = [2.0 ** -126, -2.0 ** -126, 1e-30, 2.0 ** -100, 0.9, 1.0, -3.0, 1e30, 2.0 ** 126]
SIZES = [1e-12, 2.0 ** -30, 1e-3, 8.0]  # of the gradients
READ = ["y", "u", "both"]


def check(inner, scale, size, read, x_grad=True):
    """rms without a weight as the next norm: u = y r, so that its gradient is r (du - u mean(du u))."""
    rng = np.random.default_rng(3)
    m, n, eps = 6, 20, 1e-5
    x = np.zeros((m, n), np.float32)  # the scale changes gradients alone
    f, ty, tu = (rng.standard_normal((m, n)).astype(np.float32) for _ in range(3))
    ty, tu = ty * np.float32(size), tu * np.float32(size)
    ad = A.Autodiff(inner)
    joint = A.ResidualNorm(ad, n, next=A.RMSNorm(ad, n, eps=eps), residual_scale=scale)
    tx, tf = A.Tensor.from_numpy(ad, x, requires_grad=x_grad), A.Tensor.from_numpy(ad, f, requires_grad=True)
    y, u = joint(tx, tf)
    parts = [(v * A.Tensor.from_numpy(ad, t)).sum() for v, t in ((y, ty), (u, tu)) if read in ("both", "y" if v is y else "u")]
    (parts[0] if len(parts) == 1 else parts[0] + parts[1]).backward()

    g, tol = np.zeros((m, n)), np.zeros((m, n))
    if read != "y":
        y64, t64 = f.astype(np.float64), tu.astype(np.float64)
        r = 1 / np.sqrt((y64 ** 2).mean(1, keepdims=True) + np.float64(np.float32(eps)))
        inner_sum = (t64 * y64 * r).mean(1, keepdims=True)
        g = r * (t64 - y64 * r * inner_sum)
        # sums of 20 terms over at most 17 additions; r is off by half a mean square's error and three roundings
        tol = 40 * U * r * (np.abs(t64) + np.abs(y64) * r * (np.abs(t64 * y64) * r).mean(1, keepdims=True))
    if read != "u":
        g, tol = g + ty, tol + (2 * U * (np.abs(g) + np.abs(ty)) if read == "both" else 0)
    got = y.grad().numpy()
    assert (np.abs(got - g) <= tol).all(), float(np.abs(got - g).max())
    np.testing.assert_array_equal(tf.grad().numpy(), got)  # the block's output is added as it is
    if not x_grad:
        assert tx.grad() is None
        return
    gx = tx.grad().numpy().astype(np.float64)
    want = got.astype(np.float64) * np.float64(np.float32(scale))
    # one rounding, at a float's range
    with np.errstate(over="ignore"):
        want32 = want.astype(np.float32)
    low = np.abs(want) < 2.0 ** -126  # subnormal: a multiple of 2^-149, or 0
    assert (np.abs(gx[low] - want[low]) <= np.maximum(2.0 ** -149, np.abs(want[low]))).all()
    np.testing.assert_array_equal(gx[~low], want32[~low])
