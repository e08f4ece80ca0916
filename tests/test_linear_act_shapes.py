"""LinearAct checks the shapes of its own parameters, which load_weights and optimizers replace: the product
itself sees storages and their numbers of elements only."""
from __future__ import annotations

import numpy as np
import pytest

from orcaml_amd import autodiff as A
from tests.cpu_backend import OracleBackend


class Backend(OracleBackend):
    """The CPU backend with a fused Linear that notes its calls."""
    ACTIVATIONS = {"none": 0, "relu": 1}

    def __init__(self):
        super().__init__()
        self.calls = []

    def linear_act(self, x, w, bias, residual, M, N, K, act, keep):
        self.calls.append((M, N, K))
        return self.zeros((M, N)), {}


def layer(bias=True):
    ad = A.Autodiff(Backend())
    return ad, A.LinearAct(ad, np.ones((3, 4), np.float32), np.zeros(4, np.float32) if bias else None, "relu"), \
        A.Tensor.from_numpy(ad, np.ones((2, 3), np.float32))


@pytest.mark.parametrize("shape", [(4, 3), (12,), (12, 1), (2, 6), (3, 5), (1, 3, 4)])
def test_weights_of_another_shape_are_refused(shape):
    ad, l, x = layer()
    l.weight.tensor = A.Tensor.from_numpy(ad, np.ones(shape, np.float32))
    with pytest.raises(ValueError, match="Shape mismatch during linear_act"):
        l(x)
    assert not ad.inner.calls


@pytest.mark.parametrize("shape", [(4, 1), (2, 2), (1, 5), (2, 4), (1, 1)])
def test_biases_of_another_shape_are_refused(shape):
    ad, l, x = layer()
    l.bias.tensor = A.Tensor.from_numpy(ad, np.ones(shape, np.float32))
    with pytest.raises(ValueError, match="Shape mismatch during linear_act"):
        l(x)
    assert not ad.inner.calls


def test_the_shapes_that_mean_the_same_are_taken():
    ad, l, x = layer()
    for shape in ((4,), (1, 4), (1, 1, 4)):
        l.bias.tensor = A.Tensor.from_numpy(ad, np.ones(shape, np.float32))
        assert l(x).shape == (2, 4)
    ad, l, x = layer(bias=False)
    l.weight.tensor = A.Tensor.from_numpy(ad, np.ones((4, 3), np.float32)).transpose(0, 1)
    assert l(x).shape == (2, 4) and ad.inner.calls == [(2, 4, 3)]
