"""What orca_hip_linear_act, its backward and the 8-bit checkpoints refuse, and the checkpoints'
layout: argument checks that come before any work, so they need no GPU."""
from __future__ import annotations

import ctypes

import pytest

from orcaml_amd import _lib

P = 1 << 20  # operands of the calls below: addresses that nothing reads


def _call(name, *args):
    rc = getattr(_lib.load(), name)(*args)
    return rc, _lib.load().orca_hip_last_error().decode()


def _forward(m=4, n=8, k=16, x=P, ldx=None, w=2 * P, ldw=None, y=3 * P, ldy=None, **epi):
    e = _lib.LinearEpilogue(**epi)
    return _call("orca_hip_linear_act", None, m, n, k, x, k if ldx is None else ldx, w, n if ldw is None else ldw, y,
                 n if ldy is None else ldy, ctypes.byref(e))


def _backward(m=4, n=8, k=16, dy=P, lddy=None, w=2 * P, ldw=None, dx=3 * P, lddx=None, dw=4 * P, lddw=None, db=5 * P,
              **saved):
    saved = dict(dict(x=6 * P, ldx=k), **saved)
    s = _lib.LinearSaved(**saved)
    return _call("orca_hip_linear_act_backward", None, m, n, k, dy, n if lddy is None else lddy, w,
                 n if ldw is None else ldw, ctypes.byref(s), dx, k if lddx is None else lddx, dw,
                 n if lddw is None else lddw, db)


def test_good_arguments_reach_the_context():
    for rc, msg in (_forward(), _forward(act=4, bias=7 * P, residual=8 * P, ldr=8, pre=9 * P, ldpre=9, pre8=10 * P,
                                         y8=11 * P),
                    _forward(residual=3 * P, ldr=8), _forward(ldy=24, residual=3 * P + 32, ldr=24),
                    _forward(ldy=24, residual=3 * P + 64, ldr=24), _forward(ldy=24, residual=3 * P - 32, ldr=24),
                    _forward(ldy=24, x=3 * P + 32, ldx=24), _forward(m=0, x=None, w=None, y=None), _backward(),
                    _backward(act=2, z=7 * P, ldz=8), _backward(act=2, z8=7 * P, x=None, x8=8 * P),
                    _backward(dx_add=3 * P, ldadd=16), _backward(dx_add=P, ldadd=16, k=8, ldx=8, lddx=8),
                    _backward(dx=None, w=None), _backward(dw=None, x=None), _backward(m=0, dy=None, x=None)):
        assert (rc, msg) == (_lib.ERR_INTERNAL, "null orca_hip_ctx")


@pytest.mark.parametrize("bad,code,word", [
    (dict(ldx=15), _lib.ERR_SHAPE, "(x)"), (dict(ldw=7), _lib.ERR_SHAPE, "(weight)"),
    (dict(ldy=7), _lib.ERR_SHAPE, "(y)"), (dict(residual=7 * P, ldr=7), _lib.ERR_SHAPE, "(residual)"),
    (dict(pre=7 * P, ldpre=7), _lib.ERR_SHAPE, "(pre)"), (dict(act=5), _lib.ERR_INTERNAL, "unknown activation"),
    (dict(act=-1), _lib.ERR_INTERNAL, "unknown activation"), (dict(x=None), _lib.ERR_INTERNAL, "null operand"),
    (dict(w=None), _lib.ERR_INTERNAL, "null operand"), (dict(y=None), _lib.ERR_INTERNAL, "null operand"),
    (dict(pre8=7 * P + 8), _lib.ERR_INTERNAL, "aligned"), (dict(y8=7 * P + 4), _lib.ERR_INTERNAL, "aligned"),
    (dict(y=P + 64), _lib.ERR_INTERNAL, "overlaps"), (dict(y=2 * P), _lib.ERR_INTERNAL, "overlaps"),
    (dict(pre=3 * P, ldpre=8), _lib.ERR_INTERNAL, "overlaps"), (dict(y8=3 * P), _lib.ERR_INTERNAL, "overlaps"),
    (dict(pre8=7 * P, y8=7 * P + 16), _lib.ERR_INTERNAL, "overlaps"),
    (dict(residual=3 * P, ldr=9), _lib.ERR_INTERNAL, "overlaps"),
    (dict(residual=3 * P + 4, ldr=8), _lib.ERR_INTERNAL, "overlaps"),
    (dict(pre=7 * P, ldpre=8, residual=7 * P, ldr=8), _lib.ERR_INTERNAL, "overlaps"),
    (dict(m=1 << 27), _lib.ERR_SHAPE, "2^27"), (dict(n=1 << 27), _lib.ERR_SHAPE, "2^27"),
    (dict(k=1 << 32), _lib.ERR_SHAPE, "2^27"), (dict(ldx=(1 << 34) + 1), _lib.ERR_SHAPE, "2^34"),
    (dict(ldy=24, residual=3 * P + 28, ldr=24), _lib.ERR_INTERNAL, "overlaps"),
    (dict(ldy=24, residual=3 * P + 68, ldr=24), _lib.ERR_INTERNAL, "overlaps"),
    (dict(ldy=24, residual=3 * P - 28, ldr=24), _lib.ERR_INTERNAL, "overlaps"),
    (dict(ldy=24, residual=3 * P + 32, ldr=23), _lib.ERR_INTERNAL, "overlaps")])
def test_forward_refuses(bad, code, word):
    rc, msg = _forward(**bad)
    assert rc == code and word in msg, (rc, msg)


@pytest.mark.parametrize("bad,code,word", [
    (dict(lddy=7), _lib.ERR_SHAPE, "(dy)"), (dict(ldw=7), _lib.ERR_SHAPE, "(weight)"),
    (dict(lddx=15), _lib.ERR_SHAPE, "(dx)"), (dict(lddw=7), _lib.ERR_SHAPE, "(dw)"), (dict(ldx=15), _lib.ERR_SHAPE, "(x)"),
    (dict(act=1, z=7 * P, ldz=7), _lib.ERR_SHAPE, "(z)"), (dict(dx_add=7 * P, ldadd=15), _lib.ERR_SHAPE, "(dx_add)"),
    (dict(act=9), _lib.ERR_INTERNAL, "unknown activation"), (dict(act=1), _lib.ERR_INTERNAL, "z and z8"),
    (dict(act=1, z=7 * P, ldz=8, z8=8 * P), _lib.ERR_INTERNAL, "z and z8"),
    (dict(x=None), _lib.ERR_INTERNAL, "x and x8"), (dict(x8=7 * P), _lib.ERR_INTERNAL, "x and x8"),
    (dict(dy=None), _lib.ERR_INTERNAL, "null dy"), (dict(w=None), _lib.ERR_INTERNAL, "null weight"),
    (dict(x=None, x8=7 * P + 1), _lib.ERR_INTERNAL, "aligned"),
    (dict(act=1, z8=7 * P + 1), _lib.ERR_INTERNAL, "aligned"), (dict(dx=P), _lib.ERR_INTERNAL, "overlaps"),
    (dict(dw=2 * P), _lib.ERR_INTERNAL, "overlaps"), (dict(db=4 * P), _lib.ERR_INTERNAL, "overlaps"),
    (dict(dx=6 * P), _lib.ERR_INTERNAL, "overlaps"), (dict(dx_add=3 * P, ldadd=17), _lib.ERR_INTERNAL, "overlaps"),
    (dict(dx_add=4 * P, ldadd=16), _lib.ERR_INTERNAL, "overlaps"), (dict(m=1 << 27), _lib.ERR_SHAPE, "2^27")])
def test_backward_refuses(bad, code, word):
    rc, msg = _backward(**bad)
    assert rc == code and word in msg, (rc, msg)


def _size(rows, cols):
    b, at = ctypes.c_size_t(), ctypes.c_size_t()
    _lib.call("orca_hip_act8_size", rows, cols, ctypes.byref(b), ctypes.byref(at))
    return b.value, at.value


@pytest.mark.parametrize("rows,cols,bytes_,at", [(0, 0, 0, 0), (1, 1, 32, 16), (16, 32, 528, 512), (17, 33, 576 + 64, 576),
                                                 (5, 64, 320 + 32, 320), (1 << 20, 1 << 14, (1 << 34) + (1 << 29), 1 << 34)])
def test_checkpoint_size(rows, cols, bytes_, at):
    assert _size(rows, cols) == (bytes_, at)
    b = ctypes.c_size_t()
    _lib.call("orca_hip_act8_size", rows, cols, ctypes.byref(b), None)
    assert b.value == bytes_


def test_checkpoints_refuse():
    for args, code, word in (((P, 4, 8, 7, 2 * P), _lib.ERR_SHAPE, "leading dimension"),
                             ((None, 4, 8, 8, 2 * P), _lib.ERR_INTERNAL, "null operand"),
                             ((P, 4, 8, 8, None), _lib.ERR_INTERNAL, "null operand"),
                             ((P, 4, 8, 8, 2 * P + 8), _lib.ERR_INTERNAL, "aligned"),
                             ((P, 4, 8, 8, P + 64), _lib.ERR_INTERNAL, "overlaps"),
                             ((P, 4, 8, 8, 2 * P), _lib.ERR_INTERNAL, "null orca_hip_ctx")):
        rc, msg = _call("orca_hip_act8_pack", None, *args)
        assert rc == code and word in msg, (args, rc, msg)
    for args, code, word in (((P, 4, 8, _lib.F16, 2 * P, 8), _lib.ERR_UNSUPPORTED_DTYPE, "act8_unpack"),
                             ((P, 4, 8, _lib.F32, 2 * P, 7), _lib.ERR_SHAPE, "leading dimension"),
                             ((P, 4, 8, _lib.BF16, None, 8), _lib.ERR_INTERNAL, "null operand"),
                             ((None, 4, 8, _lib.BF16, P, 8), _lib.ERR_INTERNAL, "null operand"),
                             ((P + 2, 4, 8, _lib.BF16, 2 * P, 8), _lib.ERR_INTERNAL, "aligned"),
                             ((P, 4, 8, _lib.BF16, P + 32, 8), _lib.ERR_INTERNAL, "overlaps"),
                             ((P, 4, 8, _lib.BF16, 2 * P, 8), _lib.ERR_INTERNAL, "null orca_hip_ctx")):
        rc, msg = _call("orca_hip_act8_unpack", None, *args)
        assert rc == code and word in msg, (args, rc, msg)
    for rows, cols, ld, word in ((1 << 27, 1, 1, "2^27"), (1, 1 << 27, 1 << 27, "2^27"), (1 << 40, 1 << 40, 1 << 62, "2^27"),
                                 (5, 8, 1 << 62, "2^34"), ((1 << 24) + 1, 8, 1 << 38, "2^34")):
        for fn, args in (("pack", (P, rows, cols, ld, 1 << 50)), ("unpack", (1 << 50, rows, cols, _lib.F32, P, ld))):
            rc, msg = _call("orca_hip_act8_" + fn, None, *args)
            assert rc == _lib.ERR_SHAPE and word in msg, (fn, rows, cols, ld, msg)
    rc, msg = _call("orca_hip_act8_size", 1 << 60, 1 << 60, None, None)
    assert rc == _lib.ERR_INTERNAL and "null output" in msg
    rc, msg = _call("orca_hip_act8_size", 1 << 40, 1 << 40, ctypes.byref(ctypes.c_size_t()), None)
    assert rc == _lib.ERR_SHAPE
