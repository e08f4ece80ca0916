"""A joint of no rows on the tape, and norms and dropout of no rows."""
from __future__ import annotations

import numpy as np
import pytest

from orcaml_amd import autodiff as A
from tests import residual_empty as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead,gate", E.SHAPES)
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_joint_of_no_rows(hb, lead, gate, scale):
    E.check(hb, lead, gate, scale)


@pytest.mark.parametrize("lead", [(0,), (0, 4), (4, 0)])
def test_norms_and_dropout_of_no_rows(hb, lead):
    ad = A.Autodiff(hb)
    x = A.Tensor.from_numpy(ad, np.ones((*lead, 8), np.float32), requires_grad=True)
    norm = A.LayerNorm(ad, 8, bias=np.zeros(8), checkpoint=True)
    y = A.Dropout(0.5)(norm(x))
    assert y.shape == (*lead, 8) and y.numpy().size == 0
    ad.tape.execute_backward(y.storage.node_id, hb.zeros((*lead, 8)), hb)
    assert x.grad().numpy().shape == (*lead, 8)
    for p in norm.parameters():
        np.testing.assert_array_equal(p.tensor.grad().numpy(), np.zeros((1, 8), np.float32))
