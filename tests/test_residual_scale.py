"""A joint's gradients at any residual scale, on the tape over a joint in 64 bits that rounds its results to fp32."""
from __future__ import annotations

import numpy as np
import pytest

from orcaml_amd import backend as B
from tests import norm_oracle as O
from tests import residual_scale as S
from tests.cpu_backend import OracleBackend


class Joints(OracleBackend):
    """The joint of fp32 operands without post norm, gate and dropout."""

    ResidualBlock = B.ResidualBlock
    norm = None  # a backend that has norms

    def _spec(self, b, n):
        ones, zeros = np.ones(n), np.zeros(n)
        w = ones if b.next_weight is None else b.next_weight.astype(np.float64)
        return {"post": ("none", 0.0, ones, zeros), "next": (b.next, b.next_eps, w, zeros), "gate": None,
                "rs": float(np.float32(b.residual_scale)), "bs": float(np.float32(b.block_scale)), "factor": 1.0}

    def residual_norm(self, x, f, m, n, b, checkpoint=False):
        out = O.joint(x.reshape(m, n).astype(np.float64), f.reshape(m, n).astype(np.float64), self._spec(b, n))
        return out["y"][0].astype(np.float32).reshape(-1), out["u"][0].astype(np.float32).reshape(-1), None

    def residual_norm_backward(self, dy, du, f, y, m, n, b, want=()):
        wide = lambda v: None if v is None else v.reshape(m, n).astype(np.float64)  # noqa: E731
        f = np.zeros((m, n)) if f is None else wide(f)
        out = O.joint_back(wide(dy), wide(du), f, wide(y), self._spec(b, n))
        with np.errstate(over="ignore"):
            return {k: out[k][0].astype(np.float32).reshape(-1) for k in want}


@pytest.mark.parametrize("scale", S.SCALES)
@pytest.mark.parametrize("size", S.SIZES)
@pytest.mark.parametrize("read", S.READ)
def test_gradients_at_a_scale(scale, size, read):
    S.check(Joints(), scale, size, read)
    S.check(Joints(), scale, size, read, x_grad=False)
