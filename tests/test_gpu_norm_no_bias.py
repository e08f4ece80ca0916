"""Backward kernels of norms and joints without biases, whose gradients are not asked for: each length of a row that has a
kernel, the norms that are there; and with a bias's gradient asked for of norms that have none."""
from __future__ import annotations

import pytest

from tests.test_gpu_norm import NORMS, Joint, close

pytestmark = pytest.mark.gpu

WANT = {"dx", "df", "dgate", "dpost_weight", "dnext_weight"}


def check(j, want=WANT, **sides):
    y = j.forward()["y"]
    got, oracle = j.backward(y, want=want, **sides), j.want_backward(y, **sides)
    assert got and not any(k.endswith("bias") for k in set(got) - (want - WANT))
    for k, v in got.items():
        value, tol = oracle[k]
        close(v, (value.reshape(v.shape), tol.reshape(v.shape)), (k, sides))


@pytest.mark.parametrize("n", [3, 200, 401, 1000, 1502, 3003, 6000, 8200])
@pytest.mark.parametrize("post", NORMS)
@pytest.mark.parametrize("next", NORMS)
def test_every_kernel(ctx, n, post, next):
    print(f"no bias {n} {post} {next}", flush=True)
    for groups, p in ((0, 0.1), (1, 0.0), (3, 0.0), (9, 0.3)):
        j = Joint(ctx, n + groups, 9, n, post, next, groups, p, bias=False)
        check(j)
        check(j, du=False)


# several rows a block and, with 4 and 8 waves a row, loads of the next row in flight
@pytest.mark.parametrize("m,n", [(9000, 50), (2500, 400), (5000, 700), (1500, 1500), (2000, 4096), (1100, 2600), (700, 6000)])
def test_many_rows(ctx, m, n):
    print(f"no bias {m} x {n}", flush=True)
    j = Joint(ctx, m, m, n, "layer", "rms", 1, 0.1, bias=False)
    check(j)
    check(j, dy=False)
    check(j, want=WANT | {"dnext_bias"})
    check(j, want=WANT | {"dpost_bias"})
