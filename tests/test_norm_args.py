"""What orca_hip_norm, orca_hip_residual_norm, their backward passes and orca_hip_dropout refuse: argument checks that
come before any work, so they need no GPU."""
from __future__ import annotations

import ctypes
import math

import pytest

from orcaml_amd import _lib

P = 1 << 20  # operands of the calls below: addresses that nothing reads


def _call(name, *args):
    rc = getattr(_lib.load(), name)(*args)
    return rc, _lib.load().orca_hip_last_error().decode()


def _np(kind=1, eps=1e-5, weight=None, bias=None):
    return _lib.NormParams(kind, eps, weight, bias)


def _norm(m=4, n=16, x=P, ldx=16, y=2 * P, ldy=16, y8=None, **norm):
    return _call("orca_hip_norm", None, m, n, x, ldx, ctypes.byref(_np(**norm)), y, ldy, y8)


def _norm_backward(m=4, n=16, dy=P, lddy=16, x=2 * P, ldx=16, add=None, ldadd=16, dx=3 * P, lddx=16, dw=4 * P, db=5 * P,
                   **norm):
    return _call("orca_hip_norm_backward", None, m, n, dy, lddy, x, ldx, ctypes.byref(_np(**norm)), add, ldadd, dx, lddx,
                 dw, db)


def _drop(m=4, n=16, x=P, ldx=16, p=0.5, y=2 * P, ldy=16):
    return _call("orca_hip_dropout", None, m, n, x, ldx, p, 1, 2, y, ldy)


def _block(**b):
    return _lib.ResidualBlock(**dict(dict(post=_np(2), next=_np(1), residual_scale=1.0, block_scale=1.0), **b))


def _joint(m=4, n=16, x=P, ldx=16, f=2 * P, ldf=16, y=3 * P, ldy=16, u=4 * P, ldu=16, u8=None, **b):
    return _call("orca_hip_residual_norm", None, m, n, x, ldx, f, ldf, ctypes.byref(_block(**b)), y, ldy, u, ldu, u8)


def _joint_backward(m=4, n=16, dy=P, lddy=16, du=2 * P, lddu=16, f=3 * P, ldf=16, y=4 * P, ldy=16, grads=None, **b):
    g = _lib.ResidualGrads(**(dict(dx=5 * P, lddx=16, df=6 * P, lddf=16) if grads is None else grads))
    return _call("orca_hip_residual_norm_backward", None, m, n, dy, lddy, du, lddu, f, ldf, y, ldy, ctypes.byref(_block(**b)),
                 ctypes.byref(g))


def _vectors(**more):
    return dict(dict(dx=5 * P, lddx=16, df=6 * P, lddf=16, dpost_weight=7 * P, dpost_bias=8 * P, dnext_weight=9 * P,
                     dnext_bias=10 * P), **more)


def test_good_arguments_reach_the_context():
    for rc, msg in (_norm(), _norm(kind=2, eps=0.0, weight=7 * P, bias=8 * P, y8=9 * P), _norm(y=P), _norm(m=0, x=None, y=None),
                    _norm(ldx=24, ldy=40), _norm_backward(), _norm_backward(add=3 * P), _norm_backward(dx=None, add=7 * P),
                    _norm_backward(dw=None, db=None), _norm_backward(m=0, dy=None, x=None), _drop(), _drop(p=0.0),
                    _drop(p=1.0), _drop(y=P), _joint(), _joint(y=P), _joint(next=_np(0), u=None), _joint(post=_np(0)),
                    _joint(gate=9 * P, groups=2, ldgate=16, p=0.1, u8=10 * P), _joint(m=0, x=None, f=None, y=None, u=None),
                    _joint_backward(), _joint_backward(dy=None), _joint_backward(du=None, y=None, next=_np(0)),
                    _joint_backward(du=None, y=None), _joint_backward(grads=_vectors()),
                    _joint_backward(grads=dict(dx=P, lddx=16)), _joint_backward(f=None, post=_np(0)),
                    _joint_backward(gate=12 * P, groups=4, ldgate=17, grads=_vectors(dgate=11 * P, lddgate=16)),
                    _joint_backward(m=0, dy=None, du=None, f=None, y=None)):
        assert (rc, msg) == (_lib.ERR_INTERNAL, "null orca_hip_ctx")


SHAPE, INTERNAL = _lib.ERR_SHAPE, _lib.ERR_INTERNAL


@pytest.mark.parametrize("bad,code,word", [
    (dict(ldx=15), SHAPE, "(x)"), (dict(ldy=15), SHAPE, "(y)"), (dict(kind=0), INTERNAL, "unknown norm"),
    (dict(kind=3), INTERNAL, "unknown norm"), (dict(eps=-1e-9), INTERNAL, "eps"), (dict(eps=float("nan")), INTERNAL, "eps"),
    (dict(eps=float("inf")), INTERNAL, "eps"), (dict(x=None), INTERNAL, "null operand"),
    (dict(y=None), INTERNAL, "null operand"), (dict(y8=9 * P + 8), INTERNAL, "aligned"), (dict(y=P + 64), INTERNAL, "overlaps"),
    (dict(y=P, ldy=17), INTERNAL, "overlaps"), (dict(weight=2 * P), INTERNAL, "overlaps"),
    (dict(y=P, weight=P), INTERNAL, "overlaps"), (dict(y8=2 * P), INTERNAL, "overlaps"), (dict(y8=P), INTERNAL, "overlaps"),
    (dict(m=1 << 27), SHAPE, "2^27"), (dict(n=1 << 27, ldx=1 << 27, ldy=1 << 27), SHAPE, "2^27"),
    (dict(ldx=(1 << 34) + 1), SHAPE, "2^34")])
def test_norm_refuses(bad, code, word):
    rc, msg = _norm(**bad)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("bad,code,word", [
    (dict(lddy=15), SHAPE, "(dy)"), (dict(ldx=15), SHAPE, "(x)"), (dict(lddx=15), SHAPE, "(dx)"),
    (dict(add=7 * P, ldadd=15), SHAPE, "(dx_add)"), (dict(kind=0), INTERNAL, "unknown norm"), (dict(eps=-1.0), INTERNAL, "eps"),
    (dict(dy=None), INTERNAL, "null operand"), (dict(x=None), INTERNAL, "null operand"), (dict(dx=P), INTERNAL, "overlaps"),
    (dict(dx=2 * P), INTERNAL, "overlaps"), (dict(dw=4 * P, db=4 * P + 4), INTERNAL, "overlaps"),
    (dict(dw=3 * P), INTERNAL, "overlaps"), (dict(weight=4 * P), INTERNAL, "overlaps"),
    (dict(add=3 * P, ldadd=17), INTERNAL, "overlaps"), (dict(add=5 * P), INTERNAL, "overlaps"), (dict(m=1 << 27), SHAPE, "2^27")])
def test_norm_backward_refuses(bad, code, word):
    rc, msg = _norm_backward(**bad)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("bad,code,word", [
    (dict(ldx=15), SHAPE, "(x)"), (dict(ldy=15), SHAPE, "(y)"), (dict(p=-0.1), INTERNAL, "from 0 to 1"),
    (dict(p=1.5), INTERNAL, "from 0 to 1"), (dict(p=float("nan")), INTERNAL, "from 0 to 1"), (dict(x=None), INTERNAL, "null"),
    (dict(y=None), INTERNAL, "null"), (dict(y=P + 4), INTERNAL, "overlaps"), (dict(y=P, ldy=17), INTERNAL, "overlaps"),
    (dict(n=1 << 27, ldx=1 << 27, ldy=1 << 27), SHAPE, "2^27")])
def test_dropout_refuses(bad, code, word):
    rc, msg = _drop(**bad)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("bad,code,word", [
    (dict(ldx=15), SHAPE, "(x)"), (dict(ldf=15), SHAPE, "(f)"), (dict(ldy=15), SHAPE, "(y)"), (dict(ldu=15), SHAPE, "(u)"),
    (dict(post=_np(3)), INTERNAL, "unknown norm"), (dict(next=_np(-1)), INTERNAL, "unknown norm"),
    (dict(post=_np(1, -1.0)), INTERNAL, "eps"), (dict(p=2.0), INTERNAL, "from 0 to 1"),
    (dict(gate=9 * P, groups=0, ldgate=16), SHAPE, "divides 4"), (dict(gate=9 * P, groups=3, ldgate=16), SHAPE, "divides 4"),
    (dict(gate=9 * P, groups=8, ldgate=16), SHAPE, "divides 4"), (dict(gate=9 * P, groups=2, ldgate=15), SHAPE, "(gate)"),
    (dict(x=None), INTERNAL, "null operand"), (dict(f=None), INTERNAL, "null operand"), (dict(y=None), INTERNAL, "null operand"),
    (dict(u=None), INTERNAL, "null operand"), (dict(next=_np(0)), INTERNAL, "u without"),
    (dict(next=_np(0), u=None, u8=9 * P), INTERNAL, "u without"), (dict(u8=9 * P + 4), INTERNAL, "aligned"),
    (dict(y=2 * P), INTERNAL, "overlaps"), (dict(u=P), INTERNAL, "overlaps"), (dict(u=3 * P), INTERNAL, "overlaps"),
    (dict(y=P, ldy=20), INTERNAL, "overlaps"), (dict(u8=4 * P), INTERNAL, "overlaps"),
    (dict(gate=3 * P, groups=1, ldgate=16), INTERNAL, "overlaps"), (dict(post=_np(1, weight=4 * P)), INTERNAL, "overlaps"),
    (dict(next=_np(1, bias=3 * P)), INTERNAL, "overlaps"), (dict(m=1 << 27), SHAPE, "2^27"),
    (dict(gate=9 * P, groups=1 << 40, ldgate=16, m=0), SHAPE, "divides 0")])
def test_joint_refuses(bad, code, word):
    rc, msg = _joint(**bad)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("bad,code,word", [
    (dict(lddy=15), SHAPE, "(dy)"), (dict(lddu=15), SHAPE, "(du)"), (dict(ldf=15), SHAPE, "(f)"), (dict(ldy=15), SHAPE, "(y)"),
    (dict(grads=_vectors(lddx=15)), SHAPE, "(dx)"), (dict(grads=_vectors(lddf=15)), SHAPE, "(df)"),
    (dict(gate=9 * P, groups=1, ldgate=16, grads=dict(dgate=11 * P, lddgate=15)), SHAPE, "(dgate)"),
    (dict(next=_np(0)), INTERNAL, "du without"), (dict(du=None, grads=_vectors()), INTERNAL, "need du"),
    (dict(post=_np(0), grads=_vectors()), INTERNAL, "not there"),
    (dict(grads=dict(dgate=11 * P, lddgate=16)), INTERNAL, "without its gate"),
    (dict(dy=None, du=None), INTERNAL, "one of dy and du"), (dict(f=None), INTERNAL, "null operand"),
    (dict(y=None), INTERNAL, "null operand"), (dict(p=-1.0), INTERNAL, "from 0 to 1"),
    (dict(gate=9 * P, groups=3, ldgate=16), SHAPE, "divides 4"),
    (dict(grads=_vectors(dx=P, lddx=17)), INTERNAL, "overlaps"), (dict(grads=_vectors(dx=2 * P)), INTERNAL, "overlaps"),
    (dict(grads=_vectors(df=P)), INTERNAL, "overlaps"), (dict(grads=_vectors(df=5 * P)), INTERNAL, "overlaps"),
    (dict(grads=_vectors(dpost_bias=9 * P)), INTERNAL, "overlaps"), (dict(grads=_vectors(dnext_bias=4 * P)), INTERNAL, "overlaps"),
    (dict(gate=5 * P, groups=1, ldgate=16), INTERNAL, "overlaps"), (dict(n=1 << 27), SHAPE, "2^27")])
def test_joint_backward_refuses(bad, code, word):
    rc, msg = _joint_backward(**bad)
    assert rc == code and word in msg, (rc, msg)


def test_null_parameters():
    for args in (("orca_hip_norm", None, 4, 16, P, 16, None, 2 * P, 16, None),
                 ("orca_hip_norm_backward", None, 4, 16, P, 16, 2 * P, 16, None, None, 0, 3 * P, 16, None, None),
                 ("orca_hip_residual_norm", None, 4, 16, P, 16, 2 * P, 16, None, 3 * P, 16, 4 * P, 16, None),
                 ("orca_hip_residual_norm_backward", None, 4, 16, P, 16, P, 16, P, 16, P, 16, None, None),
                 ("orca_hip_be_residual_norm", None, None, None, 4, 16, None, None, None, None),
                 ("orca_hip_be_residual_norm_backward", None, None, None, None, None, 4, 16, None) + (None,) * 7):
        rc, msg = _call(*args)
        assert rc == INTERNAL and "null parameters" in msg, msg


def test_the_rust_struct_matches_the_header():
    from tests.test_rust_binding import _c_struct, _rust_struct
    assert _rust_struct("OrcaHipBeResidualBlock") == _c_struct("orca_hip_be_residual_block")


def test_layers_need_a_backend_that_has_them():
    from orcaml_amd import autodiff as A
    ad = A.Autodiff(object())
    for layer in (A.LayerNorm, A.RMSNorm, A.ResidualNorm):
        with pytest.raises(A.OrcaError, match="needs a backend"):
            layer(ad, 4)
    x = A.Tensor(ad, A.AdStorage(None), (2, 4))
    with pytest.raises(A.OrcaError, match="needs a backend"):
        A.Dropout(0.5)(x)
    assert A.Dropout(0.5).eval()(x) is x


def test_layers_without_a_seed_draw_apart():
    from orcaml_amd import autodiff as A

    class Backend:
        residual_norm = None

    ad = A.Autodiff(Backend())
    layers = [A.Dropout(0.5), A.Dropout(0.5), A.ResidualNorm(ad, 4, p=0.5), A.ResidualNorm(ad, 4, p=0.5)]
    assert len({layer.draws.seed for layer in layers}) == len(layers)
    assert A.Dropout(0.5, seed=0).draws.seed == 0 and A.ResidualNorm(ad, 4, p=0.5, seed=7).draws.seed == 7


def test_scales_a_float_cannot_hold():
    """y's gradient is dx over the residual's scale, so the scale and its inverse are floats of full precision."""
    from orcaml_amd import autodiff as A

    class Backend:
        residual_norm = None

    ad = A.Autodiff(Backend())
    for bad in ({"residual_scale": 1e-50}, {"residual_scale": 1e-40}, {"residual_scale": -1e-40}, {"residual_scale": 1e39},
                {"residual_scale": 3e38}, {"residual_scale": 0.0}, {"residual_scale": math.nan}, {"block_scale": 1e39},
                {"block_scale": 2.0 ** 128 * (1 - 2.0 ** -30)},
                {"block_scale": -math.inf}):
        with pytest.raises(ValueError, match="scale"):
            A.ResidualNorm(ad, 4, **bad)
    for good in ({"residual_scale": 2.0 ** -126}, {"residual_scale": -2.0 ** 126}, {"block_scale": 0.0},
                 {"block_scale": 1e-50}):
        A.ResidualNorm(ad, 4, **good)


@pytest.mark.parametrize("shape,sizes", [((), (1, 1)), ((5,), (1, 5)), ((0,), (1, 0)), ((3, 0), (3, 0)), ((2, 3, 4), (6, 4))])
def test_dropout_takes_every_shape(shape, sizes):
    from orcaml_amd import autodiff as A

    class Backend:
        def dropout(self, x, rows, cols, p, seed, offset):
            assert (rows, cols) == sizes and (p, seed, offset) == (0.5, 3, 0)
            return x

    ad = A.Autodiff(Backend())
    assert A.Dropout(0.5, seed=3)(A.Tensor(ad, A.AdStorage(None), shape)).shape == shape
