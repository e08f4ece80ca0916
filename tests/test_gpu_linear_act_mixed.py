"""Models of Linear and LinearAct layers, trained with every switch of the backend and both kinds of optimizers:
an update on the second stream, a pending operand or a folded product changes no bit."""
from __future__ import annotations

import numpy as np
import pytest

from orcaml_amd import autodiff as A
from orcaml_amd.backend import HipBackend

pytestmark = pytest.mark.gpu

SWITCHES = [{}, {"overlap": True}, {"overlap": False}, {"overlap": True, "side_bpc": 2, "side_frac": 0.5}, {"lazy": False},
            {"deferred": False}, {"fold": False}]


def train(hb, optimizer, fused, checkpoint, m, d, f):
    rng = np.random.default_rng(5)
    ad = A.Autodiff(hb)

    def parameters(k, n):
        return (rng.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32), np.zeros(n, np.float32)

    layers = [A.Linear(ad, *parameters(d, f)), A.LinearAct(ad, *parameters(f, f), "gelu", checkpoint),
              A.LinearAct(ad, *parameters(f, f), "relu", checkpoint), A.Linear(ad, *parameters(f, 10))]
    params = [p for layer in layers for p in layer.parameters()]
    opt, loss = optimizer(params, lr=1e-2, fused=fused), A.CrossEntropyLoss(fused=fused)
    x = A.Tensor.from_numpy(ad, rng.standard_normal((m, d)).astype(np.float32))
    t = A.Tensor.from_numpy(ad, np.eye(10, dtype=np.float32)[rng.integers(0, 10, m)])
    out = []
    for _ in range(3):
        opt.zero_grad()
        h = layers[0](x).relu()
        h = layers[1](h, residual=h)
        h = layers[2](h, residual=h * 0.5)
        value = loss(layers[3](h), t)
        value.backward()
        opt.step()
        out.append(value.numpy())
    return out + [p.tensor.numpy() for p in params]


@pytest.mark.parametrize("m,d,f", [(64, 50, 96), (200, 130, 512)])
@pytest.mark.parametrize("optimizer", [A.AdamW, A.SGD])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_switches_change_no_bit(ctx, m, d, f, optimizer, checkpoint):
    for fused in (False, True):
        want = None
        for switches in SWITCHES:
            got = train(HipBackend(ctx, **switches), optimizer, fused, checkpoint, m, d, f)
            want = want or got
            for a, b in zip(want, got):
                np.testing.assert_array_equal(a, b, err_msg=f"{switches} fused={fused}")
