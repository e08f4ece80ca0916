"""LinearAct on the tape: a residual feed-forward block of two layers, with its activations kept in 32
and in 8 bits, against the formula in 64 bits and against differences."""
from __future__ import annotations

import gc

import numpy as np
import pytest

from orcaml_amd import _lib
from orcaml_amd import autodiff as A
from orcaml_amd.backend import Act8, HipBackend
from tests.test_gpu_linear_act import U, act64, pack64, product_tol, value64

pytestmark = pytest.mark.gpu


def block64(x, p, target, act, checkpoint):
    """Loss sum((y - t)^2) / 2 of y = act(x W1 + b1) W2 + b2 + x and its gradients, with what the
    backward reads rounded to checkpoints if `checkpoint`."""
    w1, b1, w2, b2 = (v.astype(np.float64) for v in p)
    q = (lambda v: value64(*pack64(v.astype(np.float32)))) if checkpoint else (lambda v: v)
    x = x.astype(np.float64)
    z = x @ w1 + b1
    h = act64(act, z)[0]
    y = h @ w2 + b2 + x
    g = y - target
    dh = g @ w2.T
    dz = dh * act64(act, q(z))[1]
    return (g * g).sum() / 2, {"w2": q(h).T @ g, "b2": g.sum(0, keepdims=True), "w1": q(x).T @ dz,
                               "b1": dz.sum(0, keepdims=True), "x": dz @ w1.T + g}


def problem(seed, m, d, f):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((m, d)).astype(np.float32)
    p = [(rng.uniform(-1, 1, (d, f)) / np.sqrt(d)).astype(np.float32), (rng.standard_normal((1, f)) * 0.1).astype(np.float32),
         (rng.uniform(-1, 1, (f, d)) / np.sqrt(f)).astype(np.float32), (rng.standard_normal((1, d)) * 0.1).astype(np.float32)]
    return x, p, rng.standard_normal((m, d)).astype(np.float32)


def run_block(hb, x, p, target, act, checkpoint, x_grad=True):
    ad = A.Autodiff(hb)
    l1 = A.LinearAct(ad, p[0], p[1], act, checkpoint)
    l2 = A.LinearAct(ad, p[2], p[3], "none", checkpoint)
    tx = A.Tensor.from_numpy(ad, x, requires_grad=x_grad)
    h = l1(tx)
    y = l2(h, tx)
    diff = y - A.Tensor.from_numpy(ad, target)
    loss = (diff * diff).sum() * 0.5
    loss.backward()
    grads = {"w1": l1.weight.tensor, "b1": l1.bias.tensor, "w2": l2.weight.tensor, "b2": l2.bias.tensor, "x": tx}
    return float(loss.numpy()[0]), {k: t.grad().numpy() if t.grad() is not None else None for k, t in grads.items()}, y


@pytest.mark.parametrize("m,d,f", [(1, 8, 24), (37, 50, 130), (256, 128, 512)])
@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_block_gradients(hb, m, d, f, act, checkpoint):
    x, p, target = problem(m + d + f, m, d, f)
    print(f"block {m} {d} {f} {act} {checkpoint}", flush=True)
    loss, grads, _ = run_block(hb, x, p, target, act, checkpoint)
    want_loss, want = block64(x, p, target, act, checkpoint)
    assert abs(loss - want_loss) <= 1e-4 * want_loss
    for k, g in grads.items():
        # Relative 2-norms.  In fp32: products of at most 512 terms and a chain of three, 1e-5.  With
        # checkpoints, z and h of fp32 and of 64 bits round apart where a value is within their difference
        # (below 1e-6) of the middle between two codes: with a step of 2^-7 of the group's largest value
        # at the least, about 2e-4 of the values, each by a step (below 2^-5 of the norm's share of a value):
        # sqrt(2e-4) * 2^-5 < 5e-4.
        err = np.linalg.norm(g - want[k]) / np.linalg.norm(want[k])
        assert err <= (5e-4 if checkpoint else 1e-5), (k, err)


def test_relu_block_masks(hb):
    """ReLU in fp32: the mask goes by the z that the forward computed, so values within rounding of
    zero are kept off it."""
    m, d, f = 64, 40, 96
    x, p, target = problem(3, m, d, f)
    z = x.astype(np.float64) @ p[0] + p[1]
    near = np.abs(z) < 1e-4
    assert near.mean() < 1e-3
    _, grads, _ = run_block(hb, x, p, target, "relu", False)
    _, want = block64(x, p, target, "relu", False)
    cols = ~near.any(0)
    np.testing.assert_allclose(grads["w1"][:, cols], want["w1"][:, cols], rtol=0, atol=1e-5 * np.abs(want["w1"]).max())
    np.testing.assert_allclose(grads["w2"], want["w2"], rtol=0, atol=1e-5 * np.abs(want["w2"]).max())


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_gradients_against_differences(hb, act):
    """Central differences of the device's own outputs along random directions."""
    m, d, f = 12, 20, 30
    x, p, target = problem(11, m, d, f)
    _, grads, _ = run_block(hb, x, p, target, act, False)
    rng = np.random.default_rng(5)
    for i, name in enumerate(("w1", "b1", "w2", "b2")):
        v = rng.standard_normal(p[i].shape)
        v /= np.linalg.norm(v)
        ends = []
        h = 2.0 ** -6
        for s in (1, -1):
            q = list(p)
            q[i] = (p[i] + s * h * v).astype(np.float32)
            y = run_block(hb, x, q, target, act, False)[2].numpy().astype(np.float64)
            ends.append(((y - target) ** 2).sum() / 2)
        got = (ends[0] - ends[1]) / (2 * h)
        # loss below 1e3 with y's error below 1e-6 of |y|: 1e3 * 4e-6 / 2h = 0.13; third derivatives h^2 / 6 * O(100)
        assert abs(got - float((grads[name] * v).sum())) <= 0.15 + 0.02 * abs(got), name


def test_residual_of_another_tensor_and_frozen_parts(hb):
    m, k, n = 20, 24, 36
    rng = np.random.default_rng(2)
    ad = A.Autodiff(hb)
    layer = A.LinearAct(ad, rng.standard_normal((k, n)).astype(np.float32), None, "silu")
    x = A.Tensor.from_numpy(ad, rng.standard_normal((m, k)))
    r = A.Tensor.from_numpy(ad, rng.standard_normal((m, n)), requires_grad=True)
    y = layer(x, r)
    y.sum().backward()
    np.testing.assert_array_equal(r.grad().numpy(), np.ones((m, n), np.float32))
    assert x.grad() is None and layer.weight.tensor.grad().shape == (k, n)
    # only the residual takes a gradient: nothing of the layer is kept
    layer.weight.tensor = layer.weight.tensor.detach()
    ad.tape.clear()
    layer(x, r).sum().backward()
    np.testing.assert_array_equal(r.grad().numpy(), np.ones((m, n), np.float32))
    # and none at all: no node
    ad.tape.clear()
    assert not layer(x).requires_grad and not ad.tape.nodes
    with A.no_grad(ad):
        assert not layer(x, r).requires_grad


def test_batched_input_and_transposed_operands(hb):
    rng = np.random.default_rng(4)
    ad = A.Autodiff(hb)
    w = rng.standard_normal((16, 12)).astype(np.float32)
    layer = A.LinearAct(ad, w, np.zeros(12, np.float32), "gelu")
    x = rng.standard_normal((3, 5, 16)).astype(np.float32)
    y = layer(A.Tensor.from_numpy(ad, x))
    assert y.shape == (3, 5, 12)
    xt = A.Tensor.from_numpy(ad, np.ascontiguousarray(x.reshape(15, 16).T)).transpose(0, 1)  # a lazy view
    layer.weight.tensor = A.Tensor.from_numpy(ad, np.ascontiguousarray(w.T), requires_grad=True).transpose(0, 1)
    np.testing.assert_array_equal(layer(xt).numpy(), y.numpy().reshape(15, 12))
    pending = xt.mul_scalar(2.0)  # an operand that is not computed yet
    z = 2.0 * x.reshape(15, 16).astype(np.float64) @ w
    want = act64("gelu", z)[0]
    s = 2.0 * np.abs(x.reshape(15, 16)).astype(np.float64) @ np.abs(w)
    assert (np.abs(layer(pending).numpy() - want) <= 1.2 * product_tol(s, 16) + 16 * U * np.abs(z)).all()


def test_checkpoints_take_the_memory_they_say(hb):
    """What a step keeps alive between forward and backward: the checkpoints and no activation in
    32 bits."""
    m, d, f = 1024, 256, 1024
    x, p, _ = problem(1, m, d, f)
    live = {}
    for checkpoint in (False, True):
        ad = A.Autodiff(hb)
        l1, l2 = A.LinearAct(ad, p[0], p[1], "gelu", checkpoint), A.LinearAct(ad, p[2], p[3], "none", checkpoint)
        tx = A.Tensor.from_numpy(ad, x, requires_grad=True)
        gc.collect()
        before = hb.ctx.mem_stats()["live"]
        y = l2(l1(tx), tx)
        gc.collect()
        live[checkpoint] = hb.ctx.mem_stats()["live"] - before
        del y, ad, l1, l2, tx
    assert live[False] == 4 * m * d + 2 * 4 * m * f  # y, z and h
    # The allocator's blocks: bytes in multiples of 256 up to 1 MiB, of 1 MiB from there to 16 MiB.  z and h
    # take 33 / 32 MiB as checkpoints, so 2 MiB each: 5783552 bytes with x's, y's and y itself.
    block = lambda n: -(-n // 256) * 256 if n <= 1 << 20 else -(-n // (1 << 20)) * (1 << 20)  # noqa: E731
    assert live[True] == block(4 * m * d) + 2 * block(m * f * 33 // 32) + 2 * block(m * d * 33 // 32)


def test_input_checkpoint_comes_from_the_layer_below(hb):
    x, p, _ = problem(9, 33, 40, 70)
    ad = A.Autodiff(hb)
    l1, l2 = A.LinearAct(ad, p[0], p[1], "silu", True), A.LinearAct(ad, p[2], p[3], "none", True)
    h = l1(A.Tensor.from_numpy(ad, x))
    assert isinstance(h.checkpoint, Act8) and (h.checkpoint.rows, h.checkpoint.cols) == (33, 70)
    got = hb.to_f32_vec(hb.act8_unpack(h.checkpoint)).reshape(33, 70)
    np.testing.assert_array_equal(got, value64(*pack64(h.numpy())).astype(np.float32))
    again = hb.act8_pack(h.storage.primal, 33, 70)
    np.testing.assert_array_equal(hb.to_f32_vec(hb.act8_unpack(again)).reshape(33, 70), got)
    l2(h)


def test_training_step_with_the_optimizers(hb):
    """A step through AdamW (fused and composed) moves every parameter alike."""
    x, p, target = problem(21, 96, 64, 128)
    after = []
    for fused in (False, True):
        ad = A.Autodiff(hb)
        model = A.Sequential(A.LinearAct(ad, p[0], p[1], "gelu", True), A.LinearAct(ad, p[2], p[3], "none", True))
        opt = A.AdamW(model.parameters(), lr=1e-2, fused=fused)
        tx, tt = A.Tensor.from_numpy(ad, x), A.Tensor.from_numpy(ad, target)
        for _ in range(3):
            opt.zero_grad()
            diff = model(tx) - tt
            (diff * diff).mean().backward()
            opt.step()
        after.append([q.tensor.numpy() for q in model.parameters()])
    for a, b, start in zip(*after, p):
        np.testing.assert_array_equal(a, b)
        assert not np.array_equal(a.reshape(-1), start.reshape(-1))


def test_refusals(hb):
    ad = A.Autodiff(hb)
    w = np.ones((8, 4), np.float32)
    with pytest.raises(ValueError, match="unknown activation"):
        A.LinearAct(ad, w, None, "swish")
    layer = A.LinearAct(ad, w, None, "silu")
    x = A.Tensor.from_numpy(ad, np.ones((3, 8), np.float32))
    for bad in (np.ones((3, 7), np.float32), np.ones(8, np.float32)):
        with pytest.raises(ValueError, match="Shape mismatch"):
            layer(A.Tensor.from_numpy(ad, bad))
    with pytest.raises(ValueError, match="Shape mismatch"):
        layer(x, A.Tensor.from_numpy(ad, np.ones((1, 4), np.float32)))
    with pytest.raises(ValueError, match="Device mismatch"):
        layer(x, A.Tensor.from_numpy(A.Autodiff(hb), np.ones((3, 4), np.float32)))
    s = x.storage.primal
    with pytest.raises(ValueError, match="cannot keep"):
        hb.linear_act(s, s, None, None, 3, 1, 8, keep=("z9",))
    with pytest.raises(ValueError, match="Shape mismatch"):
        hb.linear_act(s, s, None, None, 3, 4, 8)
    with pytest.raises(ValueError, match="Shape mismatch"):
        hb.linear_act_backward(s, s, 3, 8, 3, x=hb.act8_pack(s, 4, 6), want=("dw",))
    with pytest.raises(ValueError, match="cannot give"):
        hb.linear_act_backward(s, s, 3, 8, 3, want=("dz",))
    with pytest.raises(ValueError, match="z and z8"):
        hb.linear_act_backward(s, s, 3, 8, 3, "gelu", want=("dx",))


def test_another_context_is_refused(hb):
    other = HipBackend()
    s = other.from_f32_slice((3, 8), np.ones(24, np.float32))
    mine = hb.from_f32_slice((8, 4), np.ones(32, np.float32))
    with pytest.raises(ValueError, match="another context"):
        hb.linear_act(s, mine, None, None, 3, 4, 8)
    with pytest.raises(ValueError, match="another context"):
        hb.act8_unpack(other.act8_pack(s, 3, 8))


def test_fails_while_launches_go_to_the_side_stream(hb):
    s = hb.from_f32_slice((64, 64), np.ones(4096, np.float32))
    w = hb.from_f32_slice((64, 64), np.ones(4096, np.float32))
    hb.ctx.use_side_stream(1)
    try:
        with pytest.raises(ValueError, match="side stream"):
            hb.linear_act(s, w, None, None, 64, 64, 64)
    finally:
        hb.ctx.use_side_stream(0)


def test_calls_from_several_threads(hb):
    """Layers and fused optimizer passes (whose updates run on the second stream) on one backend from four threads: each
    thread's results are those of one thread."""
    import threading

    def work(seed, steps, out):
        rng = np.random.default_rng(seed)
        ad = A.Autodiff(hb)
        layers = [A.LinearAct(ad, rng.standard_normal((96, 96)).astype(np.float32) / 10, np.zeros(96, np.float32), "silu",
                              checkpoint=c) for c in (True, False)]
        opt = A.AdamW([p for layer in layers for p in layer.parameters()], lr=1e-3, fused=True)
        x = A.Tensor.from_numpy(ad, rng.standard_normal((130, 96)).astype(np.float32))
        t = A.Tensor.from_numpy(ad, rng.standard_normal((130, 96)).astype(np.float32))
        for _ in range(steps):
            opt.zero_grad()
            h = layers[0](x, residual=x)
            diff = layers[1](h, residual=h) - t
            (diff * diff).mean().backward()
            opt.step()
        out[seed] = [p.tensor.numpy() for layer in layers for p in layer.parameters()]

    alone, together = {}, {}
    for seed in range(4):
        work(seed, 6, alone)
    threads = [threading.Thread(target=work, args=(seed, 6, together)) for seed in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert sorted(together) == sorted(alone)
    for seed in alone:
        for a, b in zip(alone[seed], together[seed]):
            np.testing.assert_array_equal(a, b)


def test_refusals_of_the_calls_on_storages(hb):
    import ctypes

    s = hb.from_f32_slice((3, 8), np.ones(24, np.float32))
    w = hb.from_f32_slice((8, 4), np.ones(32, np.float32))
    out = ctypes.c_void_p()
    p = ctypes.byref(out)

    def refused(word, name, *args):
        with pytest.raises(ValueError, match=word):
            _lib.call(name, hb.handle, *args)
        assert out.value is None

    fwd, bwd = "orca_hip_be_linear_act", "orca_hip_be_linear_act_backward"
    refused("null storage", fwd, None, w.h, None, None, 3, 4, 8, 0, p, None, None, None)
    refused("null output", fwd, s.h, w.h, None, None, 3, 4, 8, 0, None, None, None, None)
    refused("Shape mismatch", fwd, s.h, w.h, None, None, 3, 4, 7, 0, p, None, None, None)
    refused("Shape mismatch", fwd, s.h, w.h, s.h, None, 3, 4, 8, 0, p, None, None, None)
    refused("Shape mismatch", fwd, s.h, w.h, None, None, 1 << 61, 4, 8, 0, p, None, None, None)
    refused("unknown activation", fwd, s.h, w.h, None, None, 3, 4, 8, 9, p, None, None, None)
    refused("one of z and z8", bwd, s.h, w.h, 3, 8, 4, 2, None, None, None, None, None, p, None, None)
    refused("one of x and x8", bwd, s.h, w.h, 3, 8, 4, 0, None, None, None, None, None, None, p, None)
    refused("Shape mismatch", bwd, s.h, w.h, 3, 8, 5, 0, None, None, None, None, None, p, None, None)
    refused("Shape mismatch", "orca_hip_be_act8_pack", s.h, 3, 9, p)
    refused("Shape mismatch", "orca_hip_be_act8_unpack", s.h, 1 << 27, 1 << 37, p)
    refused("null storage", "orca_hip_be_act8_unpack", None, 3, 8, p)
    with pytest.raises(ValueError, match="null orca_hip_backend"):
        _lib.call(fwd, None, s.h, w.h, None, None, 3, 4, 8, 0, p, None, None, None)


@pytest.mark.parametrize("m", [9, 64, 300])
def test_checkpoints_change_no_output(hb, m):
    rng = np.random.default_rng(m)
    x, w = (hb.from_f32_slice(v.shape, v) for v in (rng.standard_normal((m, 70)).astype(np.float32),
                                                    rng.standard_normal((70, 90)).astype(np.float32)))
    plain, _ = hb.linear_act(x, w, None, None, m, 90, 70, "gelu")
    y, kept = hb.linear_act(x, w, None, None, m, 90, 70, "gelu", ("z", "z8", "y8"))
    np.testing.assert_array_equal(hb.to_f32_vec(plain), hb.to_f32_vec(y))
    for k, v in (("z8", kept["z"]), ("y8", y)):  # the epilogue's checkpoints are those of its results
        np.testing.assert_array_equal(hb.to_f32_vec(hb.act8_unpack(kept[k])),
                                      hb.to_f32_vec(hb.act8_unpack(hb.act8_pack(v, m, 90))))


def test_no_rows(hb):
    x = hb.from_f32_slice((0, 8), np.zeros((0, 8), np.float32))
    w = hb.from_f32_slice((8, 4), np.ones((8, 4), np.float32))
    b = hb.from_f32_slice((1, 4), np.ones((1, 4), np.float32))
    y, kept = hb.linear_act(x, w, b, None, 0, 4, 8, "silu", ("z", "y8"))
    assert hb.to_f32_vec(y).size == 0 and hb.to_f32_vec(hb.act8_unpack(kept["y8"])).size == 0
    g = hb.linear_act_backward(y, w, 0, 4, 8, "silu", z=kept["z"], x=x)
    assert hb.to_f32_vec(g["dx"]).size == 0
    assert hb.to_f32_vec(g["dw"]).size == 32 and not np.any(hb.to_f32_vec(g["dw"]))
    assert hb.to_f32_vec(g["db"]).size == 4 and not np.any(hb.to_f32_vec(g["db"]))
