"""A joint of no rows, with each gate that its shape allows: on the CPU and on the GPU."""
from __future__ import annotations

import numpy as np

from orcaml_amd import autodiff as A

# leading dimensions of x, and of the gate (None: no gate)
SHAPES = [((0,), None), ((0,), ()), ((0,), (1,)), ((0,), (0,)), ((0, 3), (0, 3)), ((0, 3), (0, 1)), ((2, 0), (2, 0)),
          ((2, 0), (2, 1)), ((2, 0), (1, 1))]


def check(inner, lead, gate, scale):
    n, ad = 8, A.Autodiff(inner)
    leaf = lambda lead: A.Tensor.from_numpy(ad, np.ones((*lead, n), np.float32), requires_grad=True)  # noqa: E731
    joint = A.ResidualNorm(ad, n, next=A.RMSNorm(ad, n), residual_scale=scale)
    x, f, g = leaf(lead), leaf(lead), leaf(gate) if gate is not None else None
    y, u = joint(x, f, g) if g is not None else joint(x, f)
    assert y.shape == u.shape == (*lead, n) and y.numpy().size == u.numpy().size == 0
    ad.tape.execute_backward(u.storage.node_id, inner.zeros((*lead, n)), inner)
    for t in (x, f, y):
        assert t.grad().numpy().shape == (*lead, n)
    np.testing.assert_array_equal(joint.next.weight.tensor.grad().numpy(), np.zeros((1, n), np.float32))
    if g is not None:
        np.testing.assert_array_equal(g.grad().numpy(), np.zeros((*gate, n), np.float32))
