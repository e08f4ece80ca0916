"""The checkpoint that a LinearAct's output carries: taken only while it is that of the tensor's values."""
from __future__ import annotations

import gc

import numpy as np
import pytest

from orcaml_amd import autodiff as A

pytestmark = pytest.mark.gpu

M, D, F = 33, 40, 70


def layers(hb, seed=5):
    rng = np.random.default_rng(seed)
    ad = A.Autodiff(hb)
    w1, w2 = (rng.standard_normal(s).astype(np.float32) / 8 for s in ((D, F), (F, D)))
    x = A.Tensor.from_numpy(ad, rng.standard_normal((M, D)).astype(np.float32))
    return ad, A.LinearAct(ad, w1, None, "gelu", True), A.LinearAct(ad, w2, None, "silu", True), x, rng


def weight_gradient(ad, layer, x):
    ad.tape.clear()
    (layer(x) * layer(x)).sum().backward()
    return layer.weight.tensor.grad().numpy()


def by_sgd(hb, ad, s, new, rng):
    g = hb.from_f32_slice((M, F), rng.standard_normal((M, F)).astype(np.float32))
    hb.sgd_step_(s, g, M * F, 0.5)


def by_adamw(hb, ad, s, new, rng):
    g = hb.from_f32_slice((M, F), rng.standard_normal((M, F)).astype(np.float32))
    hb.adamw_step_(s, g, hb.zeros((M, F)), hb.zeros((M, F)), M * F, 0.5, 0.9, 0.999, 1e-8, 0.0, 1)


def by_one_pass(hb, ad, s, new, rng):
    g = hb.from_f32_slice((M, F), rng.standard_normal((M, F)).astype(np.float32))
    hb.sgd_multi_([(hb.clone(s), s, g, M * F)], 0.5)


def by_a_view(hb, ad, s, new, rng):
    g = hb.from_f32_slice((7, F), rng.standard_normal((7, F)).astype(np.float32))
    hb.sgd_step_(hb.view(s, 5 * F, 7 * F), g, 7 * F, 4.0)


def by_a_copy(hb, ad, s, new, rng):
    hb.copy_into(s, new.storage.primal)


@pytest.mark.parametrize("write", [by_sgd, by_adamw, by_one_pass, by_a_view, by_a_copy])
def test_values_written_in_place_leave_no_old_checkpoint(hb, write):
    """An input that is trained itself: the weight gradient is that of its present values."""
    ad, l1, l2, x, rng = layers(hb)
    h = l1(x)
    h.require_grad()
    before = weight_gradient(ad, l2, h)
    write(hb, ad, h.storage.primal, A.Tensor.from_numpy(ad, rng.standard_normal((M, F)).astype(np.float32)), rng)
    after = weight_gradient(ad, l2, h)
    np.testing.assert_array_equal(after, weight_gradient(ad, l2, A.Tensor.from_numpy(ad, h.numpy())))
    assert not np.array_equal(before, after)


def test_another_storage_leaves_no_old_checkpoint(hb):
    ad, l1, l2, x, rng = layers(hb)
    h = l1(x)
    h.storage.primal = A.Tensor.from_numpy(ad, rng.standard_normal((M, F)).astype(np.float32)).storage.primal
    np.testing.assert_array_equal(weight_gradient(ad, l2, h), weight_gradient(ad, l2, A.Tensor.from_numpy(ad, h.numpy())))


def test_the_checkpoint_is_taken_otherwise(hb):
    """No pack of its own, also for a leaf made of the output."""
    ad, l1, l2, x, _ = layers(hb)
    h = l1(x)
    packs = []
    pack, hb.act8_pack = hb.act8_pack, lambda *a: packs.append(a) or pack(*a)
    try:
        l2(h)
        h.require_grad()
        l2(h)
        assert not packs
        l2(h.detach())
        assert len(packs) == 1
    finally:
        del hb.act8_pack


def test_an_output_nobody_reads_takes_no_checkpoint(hb):
    """A last layer without its output's checkpoint: the same gradients, and its bytes less alive."""
    rng = np.random.default_rng(8)
    m, d, f = 256, 64, 128
    w1, w2 = (rng.standard_normal(s).astype(np.float32) / 8 for s in ((d, f), (f, d)))
    x = rng.standard_normal((m, d)).astype(np.float32)
    live, grads = {}, {}
    for keep in (True, False):
        ad = A.Autodiff(hb)
        l1, l2 = A.LinearAct(ad, w1, None, "gelu", True), A.LinearAct(ad, w2, None, "none", True, output_checkpoint=keep)
        tx = A.Tensor.from_numpy(ad, x)
        gc.collect()
        before = hb.ctx.mem_stats()["live"]
        y = l2(l1(tx))
        gc.collect()
        live[keep] = hb.ctx.mem_stats()["live"] - before
        assert hasattr(y, "checkpoint") == keep
        y.sum().backward()
        grads[keep] = [q.weight.tensor.grad().numpy() for q in (l1, l2)]
        del y, ad, l1, l2, tx
    assert live[True] - live[False] == m * d * 33 // 32  # a multiple of the allocator's 256 bytes
    for a, b in zip(grads[True], grads[False]):
        np.testing.assert_array_equal(a, b)
