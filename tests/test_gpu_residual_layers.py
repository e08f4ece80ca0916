"""LayerNorm, RMSNorm, Dropout and ResidualNorm on the tape: each against the formulas in 64 bits, and a run of two
residual feed-forward blocks with all of them against the formula and against differences."""
from __future__ import annotations

import gc

import numpy as np
import pytest

from orcaml_amd import autodiff as A
from orcaml_amd.backend import Act8, HipBackend
from tests import norm_oracle as O
from tests.norm_oracle import U
from tests.test_gpu_linear_act import act64
from tests.test_gpu_norm import EPS, close, stream

pytestmark = pytest.mark.gpu


def vec(rng, n, mean):
    return (mean + 0.3 * rng.standard_normal(n)).astype(np.float32)


@pytest.mark.parametrize("cls,kind", [(A.LayerNorm, "layer"), (A.RMSNorm, "rms")])
@pytest.mark.parametrize("shape", [(24,), (7, 100), (3, 5, 33)])
@pytest.mark.parametrize("bias", [True, False])
def test_norms(hb, cls, kind, shape, bias):
    rng = np.random.default_rng(sum(shape))
    n, m = shape[-1], int(np.prod(shape[:-1]))
    ad = A.Autodiff(hb)
    x, w, b, t = stream(rng, m, n), vec(rng, n, 1), vec(rng, n, 0) if bias else None, stream(rng, m, n)
    layer = cls(ad, n, w, b)
    tx = A.Tensor.from_numpy(ad, x.reshape(shape), requires_grad=True)
    y = layer(tx)
    assert y.shape == shape
    b64 = b.astype(np.float64) if bias else np.zeros(n)
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    close(y.numpy().reshape(m, n), O.norm(kind, x64, EPS, w64, b64), "y")
    (y * A.Tensor.from_numpy(ad, t.reshape(shape))).sum().backward()
    (d, td), (vw, tw), (vb, tb) = O.norm_back(kind, x64, EPS, w64, t.astype(np.float64))
    close(tx.grad().numpy().reshape(m, n), (d, td), "dx")
    close(layer.weight.tensor.grad().numpy(), (vw[None], tw[None]), "dw")
    if bias:
        close(layer.bias.tensor.grad().numpy(), (vb[None], tb[None]), "db")


def test_norm_of_frozen_parts(hb):
    ad = A.Autodiff(hb)
    layer = A.LayerNorm(ad, 16, bias=np.zeros(16))
    x = A.Tensor.from_numpy(ad, np.random.default_rng(0).standard_normal((4, 16)), requires_grad=True)
    layer.weight.tensor = layer.weight.tensor.detach()
    layer(x).sum().backward()
    assert layer.weight.tensor.grad() is None and layer.bias.tensor.grad().shape == (1, 16) and x.grad().shape == (4, 16)
    layer.bias.tensor = layer.bias.tensor.detach()
    ad.tape.clear()
    assert not layer(x.detach()).requires_grad and not ad.tape.nodes
    with A.no_grad(ad):
        assert not layer(x).requires_grad


def test_dropout_layer(hb):
    ad = A.Autodiff(hb)
    rng = np.random.default_rng(1)
    x, t = rng.standard_normal((6, 5, 21)).astype(np.float32), rng.standard_normal((6, 5, 21)).astype(np.float32)
    drop = A.Dropout(0.3, seed=1 << 40)
    tx = A.Tensor.from_numpy(ad, x, requires_grad=True)
    for call in range(3):
        ad.tape.clear()
        y = drop(tx)
        factor = O.dropout_factor(30, 21, 0.3, 1 << 40, call).reshape(x.shape)
        np.testing.assert_allclose(y.numpy(), x * factor, rtol=3 * U, atol=0)
        (y * A.Tensor.from_numpy(ad, t)).sum().backward()
        np.testing.assert_allclose(tx.grad().numpy(), t * factor, rtol=3 * U, atol=0)
    again = A.Dropout(0.3, seed=1 << 40)
    np.testing.assert_array_equal(again(tx).numpy() == 0, O.dropout_factor(30, 21, 0.3, 1 << 40, 0).reshape(x.shape) == 0)
    assert drop.eval()(tx) is tx and A.Dropout(0.0)(tx) is tx
    assert drop.train().draws.calls == 3
    assert (A.Dropout(1.0)(tx).numpy() == 0).all()
    ad.tape.clear()
    assert not drop(tx.detach()).requires_grad and not ad.tape.nodes


def test_train_and_eval_reach_every_module():
    model = A.Sequential(A.Dropout(0.5), A.Sequential(A.ReLU(), A.Dropout(0.1)))
    assert all(m.training for m in (model, *model._modules.values()))
    assert model.eval() is model
    inner = list(model._modules.values())[1]
    assert not any(m.training for m in (model, inner, *inner._modules.values()))
    model.train()
    assert inner._modules["1"].training


@pytest.mark.parametrize("post,nxt", [(None, None), ("rms", None), (None, "layer"), ("layer", "rms")])
@pytest.mark.parametrize("gate", [None, "own", "rows", "groups", "one"])
def test_joint(hb, post, nxt, gate):
    rng = np.random.default_rng(len(str((post, nxt, gate))))
    n, lead = 45, (4, 6)
    m, ad = 24, A.Autodiff(hb)
    cls = {"layer": A.LayerNorm, "rms": A.RMSNorm}
    vectors = {k: vec(rng, n, i % 2 == 0) for i, k in enumerate(("post_w", "post_b", "next_w", "next_b"))}
    own = vec(rng, n, 0.7) if gate == "own" else None
    joint = A.ResidualNorm(ad, n, cls[post](ad, n, vectors["post_w"], vectors["post_b"]) if post else None,
                           cls[nxt](ad, n, vectors["next_w"], vectors["next_b"]) if nxt else None, own, p=0.25, seed=77,
                           residual_scale=0.5, block_scale=2.0)
    x, f, ty, tu = (stream(rng, m, n) for _ in range(4))
    rows = {"rows": lead, "groups": (4, 1), "one": ()}.get(gate)
    g = stream(rng, max(1, int(np.prod(rows))), n) if rows is not None else own.reshape(1, n) if gate else None
    leaf = lambda v, lead: A.Tensor.from_numpy(ad, v.reshape(*lead, n), requires_grad=True)  # noqa: E731
    tx, tf = leaf(x, lead), leaf(f, lead)
    tg = leaf(g, rows) if rows is not None else None
    out = joint(tx, tf, tg) if tg is not None else joint(tx, tf)
    y, u = out if nxt else (out, None)
    d64 = lambda v: v.astype(np.float64)  # noqa: E731
    spec = {"post": (post or "none", EPS, d64(vectors["post_w"]), d64(vectors["post_b"])),
            "next": (nxt or "none", EPS, d64(vectors["next_w"]), d64(vectors["next_b"])),
            "gate": d64(g) if g is not None else None, "rs": 0.5, "bs": 2.0,
            "factor": O.dropout_factor(m, n, 0.25, 77, 0)}
    want = O.joint(d64(x), d64(f), spec)
    close(y.numpy().reshape(m, n), want["y"], "y")
    loss = (y * A.Tensor.from_numpy(ad, ty.reshape(*lead, n))).sum()
    if u is not None:
        close(u.numpy().reshape(m, n), want["u"], "u")
        loss = loss + (u * A.Tensor.from_numpy(ad, tu.reshape(*lead, n))).sum()
    loss.backward()
    back = O.joint_back(d64(ty), d64(tu) if nxt else None, d64(f), d64(y.numpy().reshape(m, n)), spec)
    got = {"dx": tx, "df": tf}
    if gate:
        got["dgate"] = joint.gate.tensor if gate == "own" else tg
    for name, norm in (("post", joint.post), ("next", joint.next)):
        if norm is not None:
            got |= {f"d{name}_weight": norm.weight.tensor, f"d{name}_bias": norm.bias.tensor}
    for k, t in got.items():
        v = t.grad().numpy().reshape(-1, n)
        close(v, tuple(np.broadcast_to(b, back[k][0].shape).reshape(v.shape) for b in back[k]), k)
    # y's own gradient, with what came through u
    v, tol = back["dx"]
    close(y.grad().numpy().reshape(m, n), (v / 0.5, tol / 0.5 + 2 * U * np.abs(v / 0.5)), "y.grad()")


def test_joint_with_one_side_unread(hb):
    rng = np.random.default_rng(3)
    x, f = rng.standard_normal((8, 20)), rng.standard_normal((8, 20))
    for read in ("y", "u"):
        ad = A.Autodiff(hb)
        joint = A.ResidualNorm(ad, 20, next=A.RMSNorm(ad, 20))
        tx, tf = (A.Tensor.from_numpy(ad, v, requires_grad=True) for v in (x, f))
        y, u = joint(tx, tf)
        (y if read == "y" else u).sum().backward()
        if read == "y":
            np.testing.assert_array_equal(tx.grad().numpy(), np.ones((8, 20), np.float32))
            assert joint.next.weight.tensor.grad() is None
        else:
            assert joint.next.weight.tensor.grad().shape == (1, 20)
            np.testing.assert_array_equal(tx.grad().numpy(), tf.grad().numpy())
    ad.tape.clear()
    y, u = joint(tx, tf)
    ad.tape.execute_backward(A.Tensor.from_numpy(ad, [1.0], True).storage.node_id, None, hb)  # nothing of the joint
    assert tx.grad() is None


def test_joint_of_one_tensor_and_itself(hb):
    """x as the stream and as the block's output: its gradient is the sum of both."""
    ad = A.Autodiff(hb)
    x = np.random.default_rng(5).standard_normal((3, 12)).astype(np.float32)
    tx = A.Tensor.from_numpy(ad, x, requires_grad=True)
    y = A.ResidualNorm(ad, 12, block_scale=3.0)(tx, tx)
    np.testing.assert_array_equal(y.numpy(), x + 3 * x)
    y.sum().backward()
    np.testing.assert_array_equal(tx.grad().numpy(), np.full((3, 12), 4, np.float32))


def test_joint_in_evaluation(hb):
    ad = A.Autodiff(hb)
    rng = np.random.default_rng(6)
    x, f = (A.Tensor.from_numpy(ad, rng.standard_normal((5, 16))) for _ in range(2))
    joint = A.ResidualNorm(ad, 16, p=0.5)
    assert (joint(x, f).numpy() != (x + f).numpy()).any()
    np.testing.assert_array_equal(joint.eval()(x, f).numpy(), (x + f).numpy())
    assert joint.draws.calls == 1


def test_checkpoints_go_on_to_the_layer_above(hb):
    ad = A.Autodiff(hb)
    rng = np.random.default_rng(7)
    up = A.LinearAct(ad, rng.standard_normal((40, 64)).astype(np.float32) / 6, None, "gelu", checkpoint=True)
    x, f = (A.Tensor.from_numpy(ad, rng.standard_normal((50, 40)), requires_grad=True) for _ in range(2))
    norm = A.LayerNorm(ad, 40, checkpoint=True)
    joint = A.ResidualNorm(ad, 40, next=A.RMSNorm(ad, 40, checkpoint=True))
    for u in (norm(x), joint(x, f)[1]):
        assert isinstance(u.checkpoint, Act8) and A.LinearAct._checkpoint_of(u) is u.checkpoint
        mine, packed = hb.act8_unpack(u.checkpoint), hb.act8_unpack(hb.act8_pack(u.storage.primal, 50, 40))
        np.testing.assert_array_equal(hb.to_f32_vec(mine), hb.to_f32_vec(packed))
        up(u).sum().backward()
    with A.no_grad(ad):  # nothing to keep
        assert not hasattr(norm(x), "checkpoint")


def test_the_joint_keeps_what_its_backward_reads(hb):
    """Without post norm and gate nothing of f is kept, without a next norm nothing of y."""
    m, n = 512, 1024
    ad = A.Autodiff(hb)
    for post, nxt, kept in ((None, None, 0), ("rms", None, 1), (None, "rms", 1), ("rms", "rms", 2)):
        joint = A.ResidualNorm(ad, n, A.RMSNorm(ad, n) if post else None, A.RMSNorm(ad, n) if nxt else None, p=0.1)
        ad.tape.clear()
        x = A.Tensor.from_numpy(ad, np.zeros((m, n)), requires_grad=True)
        gc.collect()
        before = hb.ctx.mem_stats()["live"]
        f = A.Tensor.from_numpy(ad, np.ones((m, n)), requires_grad=True)
        out = joint(x, f)
        del f, out
        gc.collect()
        assert hb.ctx.mem_stats()["live"] - before == kept * 4 * m * n
        del x
    ad.tape.clear()


def test_nodes_hold_no_cycle(hb):
    """A tape that is dropped releases its storages at once."""
    gc.collect()
    gc.disable()
    try:
        before = hb.ctx.mem_stats()["live"]
        ad = A.Autodiff(hb)
        x, f = (A.Tensor.from_numpy(ad, np.ones((64, 128)), requires_grad=True) for _ in range(2))
        joint = A.ResidualNorm(ad, 128, A.RMSNorm(ad, 128), A.LayerNorm(ad, 128), p=0.1)
        y, u = joint(A.Dropout(0.5)(A.LayerNorm(ad, 128)(x)), f)
        (y.sum() + u.sum()).backward()
        assert hb.ctx.mem_stats()["live"] > before
        del ad, x, f, joint, y, u
        assert hb.ctx.mem_stats()["live"] == before
    finally:
        gc.enable()


class Block:
    """norm, up, down, joint: two residual feed-forward blocks with everything there is."""

    def __init__(self, hb, d, f, checkpoint=False):
        self.ad = A.Autodiff(hb)
        rng = np.random.default_rng(d + f)
        ad = self.ad
        self.norm = A.LayerNorm(ad, d, vec(rng, d, 1), vec(rng, d, 0), checkpoint=checkpoint)
        self.ff, self.joints, modules = [], [], [self.norm]
        for i in range(2):
            up = A.LinearAct(ad, (rng.standard_normal((d, f)) / np.sqrt(d)).astype(np.float32), vec(rng, f, 0), "gelu", checkpoint)
            down = A.LinearAct(ad, (rng.standard_normal((f, d)) / np.sqrt(f)).astype(np.float32), None, "none", checkpoint)
            joint = A.ResidualNorm(ad, d, A.RMSNorm(ad, d, vec(rng, d, 1)),
                                   A.LayerNorm(ad, d, vec(rng, d, 1), vec(rng, d, 0), checkpoint=checkpoint),
                                   gate_weight=vec(rng, d, 0.5) if i else None, p=0.1, seed=100 + i, residual_scale=0.9)
            self.ff.append((up, down))
            self.joints.append(joint)
            modules += [up, down, joint]
        self.model = A.Sequential(*modules)

    def __call__(self, x, gate):
        u = self.norm(x)
        for i, ((up, down), joint) in enumerate(zip(self.ff, self.joints)):
            x, u = joint(x, down(up(u)), gate) if i == 0 else joint(x, down(up(u)))
        return x, u

    def rewind(self):
        """The next run draws the first one's numbers again."""
        for j in self.joints:
            j.draws.calls = 0


def run64(b, x, gate, p):
    """(x, u) in 64 bits with parameters p: [norm w, b, up w, b, down w, (gate), post w, next w, b, ...]."""
    p = iter(p)
    d = x.shape[1]
    u = O.norm("layer", x, EPS, next(p).reshape(-1), next(p).reshape(-1))[0]
    for i in range(2):
        wu, bu, wd = next(p), next(p), next(p)
        own = next(p) if i else gate
        post, nw, nb = next(p), next(p), next(p)
        f = act64("gelu", u @ wu + bu)[0] @ wd
        out = O.joint(x, f, {"post": ("rms", EPS, post.reshape(-1), np.zeros(d)),
                             "next": ("layer", EPS, nw.reshape(-1), nb.reshape(-1)), "gate": own, "rs": float(np.float32(0.9)),
                             "bs": 1.0, "factor": O.dropout_factor(x.shape[0], d, 0.1, 100 + i, 0)})
        x, u = out["y"][0], out["u"][0]
    return x, u


@pytest.mark.parametrize("m,d,f", [(8, 24, 48), (96, 130, 200)])
def test_two_blocks(hb, m, d, f):
    rng = np.random.default_rng(m)
    x, gate, tx, tu = stream(rng, m, d, 0.0), vec(rng, 4 * d, 0.8).reshape(4, d), stream(rng, m, d), stream(rng, m, d)
    b = Block(hb, d, f)
    tensors = [A.Tensor.from_numpy(b.ad, v, requires_grad=True) for v in (x, gate)]
    y, u = b(*tensors)
    params = [p.tensor for p in b.model.parameters()]
    # order of a joint's parameters: its own gate, then its norms'
    host = [t.numpy().astype(np.float64) for t in params]
    want = run64(b, x.astype(np.float64), gate.astype(np.float64), host)
    # a chain of some twenty operators, each a few hundred roundings wide at the most and about 1 in size
    for got, w in zip((y, u), want):
        assert np.linalg.norm(got.numpy() - w) <= 1e-5 * np.linalg.norm(w)
    loss = (y * A.Tensor.from_numpy(b.ad, tx)).sum() + (u * A.Tensor.from_numpy(b.ad, tu)).sum()
    loss.backward()

    def loss64(values):
        yy, uu = run64(b, values[0], values[1], values[2:])
        return (yy * tx).sum() + (uu * tu).sum()

    values = [x.astype(np.float64), gate.astype(np.float64), *host]
    for i, t in enumerate([*tensors, *params]):
        g = t.grad().numpy().astype(np.float64)
        v = rng.standard_normal(values[i].shape)
        v /= np.linalg.norm(v)
        h = 1e-4
        ends = [loss64([w + s * h * v if k == i else w for k, w in enumerate(values)]) for s in (1, -1)]
        got = float((g.reshape(v.shape) * v).sum())
        # differences in 64 bits: h^2 / 6 times third derivatives (about |g|), and 1e-16 of the loss over h; the
        # gradient's own error as that of the values above
        assert abs(got - (ends[0] - ends[1]) / (2 * h)) <= 2e-5 * np.linalg.norm(g) + 1e-7, i


def test_training_steps_with_the_optimizers(hb):
    """Steps through AdamW, fused and composed, move every parameter alike, and repeat from the seeds."""
    rng = np.random.default_rng(9)
    x, t = stream(rng, 64, 48, 0.0), stream(rng, 64, 48)
    after = []
    for fused in (False, True, True):
        b = Block(hb, 48, 96, checkpoint=True)
        opt = A.AdamW(b.model.parameters(), lr=1e-2, fused=fused)
        tx, tt = A.Tensor.from_numpy(b.ad, x), A.Tensor.from_numpy(b.ad, t)
        for _ in range(3):
            opt.zero_grad()
            y, u = b(tx, A.Tensor.from_numpy(b.ad, np.ones((1, 48))))
            diff = u - tt
            ((diff * diff).mean() + (y * y).mean()).backward()
            opt.step()
        after.append([p.tensor.numpy() for p in b.model.parameters()])
    start = [p.tensor.numpy() for p in Block(hb, 48, 96).model.parameters()]
    for a, c, e, s in zip(*after, start):
        np.testing.assert_array_equal(a, c)
        np.testing.assert_array_equal(c, e)
        assert not np.array_equal(a, s)


def test_weights_are_saved_and_loaded(hb, tmp_path):
    a, b = Block(hb, 24, 40), Block(hb, 24, 40)
    for p in b.model.parameters():
        p.tensor = A.Tensor.zeros(b.ad, p.tensor.shape, requires_grad=True)
    a.model.save_weights(str(tmp_path / "w.safetensors"))
    b.model.load_weights(str(tmp_path / "w.safetensors"))
    rng = np.random.default_rng(2)
    x, gate = stream(rng, 6, 24), stream(rng, 1, 24)
    outs = [m(A.Tensor.from_numpy(m.ad, x), A.Tensor.from_numpy(m.ad, gate))[1].numpy() for m in (a, b)]
    np.testing.assert_array_equal(*outs)


def test_refusals(hb):
    ad, other = A.Autodiff(hb), A.Autodiff(hb)
    ones = lambda *s: A.Tensor.from_numpy(ad, np.ones(s))  # noqa: E731
    norm = A.LayerNorm(ad, 8)
    for bad in (ones(3, 7), ones(9)):
        with pytest.raises(ValueError, match="Shape mismatch"):
            norm(bad)
    with pytest.raises(ValueError, match="Device mismatch"):
        norm(A.Tensor.from_numpy(other, np.ones((3, 8))))
    norm.weight.tensor = ones(8, 1)
    with pytest.raises(ValueError, match="Shape mismatch"):
        norm(ones(3, 8))
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="from 0 to 1"):
            A.Dropout(p)
        with pytest.raises(ValueError, match="from 0 to 1"):
            A.ResidualNorm(ad, 8, p=p)
    for seed in (-1, 2 ** 64):
        with pytest.raises(ValueError, match="64 bits"):
            A.Dropout(0.5, seed=seed)
        with pytest.raises(ValueError, match="64 bits"):
            hb.dropout(ones(3, 8).storage.primal, 3, 8, 0.5, 0, seed)
    for scales in ({"residual_scale": 0.0}, {"residual_scale": float("inf")}, {"block_scale": float("nan")}):
        with pytest.raises(ValueError, match="scales"):
            A.ResidualNorm(ad, 8, **scales)
    with pytest.raises(ValueError, match="Shape mismatch"):
        A.ResidualNorm(ad, 8, post=A.RMSNorm(ad, 9))
    joint = A.ResidualNorm(ad, 8)
    for x, f, g in ((ones(6, 8), ones(6, 7), None), (ones(6, 8), ones(3, 8), None), (ones(6, 8), ones(6, 8), ones(4, 8)),
                    (ones(6, 8), ones(6, 8), ones(6, 7)), (ones(6, 7), ones(6, 7), None),
                    (ones(4, 6, 8), ones(4, 6, 8), ones(1, 6, 8)), (ones(4, 4, 8), ones(4, 4, 8), ones(4, 8)),
                    (ones(4, 6, 8), ones(4, 6, 8), ones(2, 1, 8))):
        with pytest.raises(ValueError, match="Shape mismatch"):
            joint(x, f, g)
    with pytest.raises(ValueError, match="no other|takes no"):
        A.ResidualNorm(ad, 8, gate_weight=np.ones(8))(ones(6, 8), ones(6, 8), ones(6, 8))
    with pytest.raises(ValueError, match="Device mismatch"):
        joint(ones(6, 8), A.Tensor.from_numpy(other, np.ones((6, 8))))
    s = ones(3, 8).storage.primal
    with pytest.raises(ValueError, match="unknown norm"):
        hb.norm(s, 3, 8, "batch")
    with pytest.raises(ValueError, match="Shape mismatch"):
        hb.norm(s, 3, 9, "rms")
    with pytest.raises(ValueError, match="unknown norm"):
        hb.norm(s, 3, 8, "none")
    with pytest.raises(ValueError, match="cannot give"):
        hb.norm_backward(s, s, 3, 8, "rms", want=("dy",))
    with pytest.raises(ValueError, match="without its gate"):
        hb.residual_norm_backward(s, None, s, s, 3, 8, hb.ResidualBlock(), want=("dgate",))
    with pytest.raises(ValueError, match="one of dy and du"):
        hb.residual_norm_backward(None, None, s, s, 3, 8, hb.ResidualBlock())
    mine = HipBackend()
    with pytest.raises(ValueError, match="another context"):
        mine.norm(s, 3, 8, "rms")


def test_pending_and_transposed_operands(hb):
    """A chain that is not computed yet, and a lazy transpose, as operands."""
    ad = A.Autodiff(hb)
    x = np.random.default_rng(8).standard_normal((12, 20)).astype(np.float32)
    tx = A.Tensor.from_numpy(ad, np.ascontiguousarray(x.T)).transpose(0, 1)
    norm = A.RMSNorm(ad, 20)
    want = norm(A.Tensor.from_numpy(ad, x)).numpy()
    np.testing.assert_array_equal(norm(tx).numpy(), want)
    twice = A.Tensor.from_numpy(ad, x).mul_scalar(2.0)
    np.testing.assert_array_equal(A.ResidualNorm(ad, 20)(twice, twice).numpy(), x * 4)
