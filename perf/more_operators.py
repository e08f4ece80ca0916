"""The ends of a residual block, as measurable cases: norms of rows, dropout, and the joint of one block with the next.

  norm_fwd   y = norm(x) w + b of each row, by mean and variance ("layer") or by the mean square ("rms"); it may keep
             y's 8-bit checkpoint as well
  norm_bwd   dx (with the gradient that came past the norm added), dw and db from dy and x
  join_fwd   y = s x + t gate * drop(post(f)): a block's output f, normed, thinned out, gated and added to the stream
             x; and u = next(y), the next block's input
  join_bwd   dx, df, dgate and the gradients of both norms' weights from dy, du, f and y
  drop       y = x / (1 - p) where a random number says so, else 0; dx from dy is the same pass

A value's random number is word col % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011) at the counter
(col / 4, row, offset, offset >> 32) under the key (seed, seed >> 32): it is kept where that is at least
rint(p 2^32).  A gate has `groups` rows, each for as many successive rows of f: one row for all (a scale a channel),
one a sample, or one a row.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

NORMS = ("none", "layer", "rms")
EPS = 1e-5


def listed():
    return [
        # the last norm before a classifier for one sample, as a service asks for it: latency
        {"name": "norm_fwd_one_row", "kind": "norm_fwd", "rows": 1, "cols": 4096, "norm": "rms", "bias": False,
         "keep8": False},
        # before the hidden layer of the benchmark's configuration, whose input is kept in 8 bits
        {"name": "norm_fwd_8bit", "kind": "norm_fwd", "rows": 1024, "cols": 4096, "norm": "layer", "bias": True,
         "keep8": True},
        # the middle configuration's hidden width
        {"name": "norm_bwd_medium", "kind": "norm_bwd", "rows": 256, "cols": 1024, "norm": "layer", "bias": True,
         "add": False},
        # a large batch, with the gradient that came past the block
        {"name": "norm_bwd_large", "kind": "norm_bwd", "rows": 8192, "cols": 4096, "norm": "rms", "bias": False,
         "add": True},
        # the smallest configuration: dropout, addition and the next block's norm
        {"name": "join_fwd_small", "kind": "join_fwd", "rows": 64, "cols": 128, "post": "none", "next": "layer",
         "bias": True, "groups": 0, "p": 0.1, "scaled": False},
        # an odd width and the last, partial batch of an epoch; a gate of its own for each value
        {"name": "join_fwd_ragged", "kind": "join_fwd", "rows": 777, "cols": 1003, "post": "layer", "next": "layer",
         "bias": True, "groups": 777, "p": 0.2, "scaled": True},
        # a large batch: both norms, a scale a channel, dropout
        {"name": "join_fwd_large", "kind": "join_fwd", "rows": 8192, "cols": 4096, "post": "rms", "next": "rms",
         "bias": False, "groups": 1, "p": 0.1, "scaled": False},
        # 32 samples of 64 rows, each with a gate from its own conditions
        {"name": "join_bwd_groups", "kind": "join_bwd", "rows": 2048, "cols": 1024, "post": "none", "next": "layer",
         "bias": True, "groups": 32, "p": 0.0, "scaled": False},
        # odd sizes, training, everything there is
        {"name": "join_bwd_ragged", "kind": "join_bwd", "rows": 777, "cols": 1501, "post": "layer", "next": "layer",
         "bias": True, "groups": 777, "p": 0.2, "scaled": True},
        # the large batch's backward
        {"name": "join_bwd_large", "kind": "join_bwd", "rows": 8192, "cols": 4096, "post": "rms", "next": "rms",
         "bias": False, "groups": 1, "p": 0.1, "scaled": False},
        # a small network's input: launches
        {"name": "drop_small", "kind": "drop", "rows": 64, "cols": 784, "p": 0.2},
        # the activation of a large batch, or its gradient: memory
        {"name": "drop_large", "kind": "drop", "rows": 8192, "cols": 4096, "p": 0.1},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over the logarithm; about half are multiples of 8."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 8:
        n = n // 8 * 8
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(["norm_fwd", "norm_bwd", "join_fwd", "join_fwd", "join_bwd", "join_bwd", "drop"])
    cols = _size(rng, 8, 8192)
    rows = _size(rng, 1, min(8192, 2 ** 25 // cols))
    case = {"kind": kind, "rows": rows, "cols": cols}
    if kind in ("norm_fwd", "norm_bwd"):
        case |= {"norm": rng.choice(NORMS[1:]), "bias": rng.random() < 0.5}
        case |= {"keep8": rng.random() < 0.3} if kind == "norm_fwd" else {"add": rng.random() < 0.5}
    elif kind == "drop":
        case["p"] = rng.choice([0.05, 0.1, 0.3, 0.5])
    else:
        groups = rng.choice([0, 1, rows, "some"])
        if groups == "some":
            groups = rng.choice([g for g in range(1, rows + 1) if rows % g == 0])
        case |= {"post": rng.choice(NORMS), "next": rng.choice(NORMS), "bias": rng.random() < 0.5, "groups": groups,
                 "p": rng.choice([0.0, 0.1, 0.3]), "scaled": rng.random() < 0.3}
    return case


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _stream(g, rows, cols):
    """A residual stream: channels of unequal size and mean, rows of unequal size."""
    return (_normal(g, (rows, cols)) + _normal(g, (1, cols), 0.3)) * torch.exp(_normal(g, (1, cols), 0.5)) \
        * torch.exp(_normal(g, (rows, 1), 0.3))


def _weights(t, g, name, kind, cols, bias):
    if kind != "none":
        t[name + "_w"] = 1 + _normal(g, (cols,), 0.2)
        if bias:
            t[name + "_b"] = _normal(g, (cols,), 0.1)


def _inputs(case, seed):
    g, m, n = _gen(seed), case["rows"], case["cols"]
    kind = case["kind"]
    if kind == "drop":
        return {"x": _normal(g, (m, n))}
    t = {}
    if kind in ("norm_fwd", "norm_bwd"):
        t["x"] = _stream(g, m, n)
        _weights(t, g, "norm", case["norm"], n, case["bias"])
        if kind == "norm_bwd":
            t["dy"] = _normal(g, (m, n), 1.0 / m)
            if case["add"]:
                t["add"] = _normal(g, (m, n), 1.0 / m)
        return t
    t["f"] = _normal(g, (m, n)) * torch.exp(_normal(g, (1, n), 0.3))
    _weights(t, g, "post", case["post"], n, case["bias"])
    _weights(t, g, "next", case["next"], n, case["bias"])
    if case["groups"]:
        t["gate"] = 0.7 + _normal(g, (case["groups"], n), 0.3)
    t["x" if kind == "join_fwd" else "y"] = _stream(g, m, n)
    if kind == "join_bwd":
        t["dy"] = _normal(g, (m, n), 1.0 / m)
        if case["next"] != "none":
            t["du"] = _normal(g, (m, n), 1.0 / m)
    return t


def _noise(seed):
    """The dropout's seed and offset of a run: numbers of 64 bits that depend on the run."""
    a = (int(seed) * 0x9E3779B97F4A7C15 + 0x632BE59BD9B4E019) % 2 ** 64
    return a, (a >> 7) * 3 % 2 ** 64


def _scales(case):
    return (0.81, 1.25) if case["scaled"] else (1.0, 1.0)


_ctx = None


def prepare(case, seed):
    """The inputs, and the buffers that a program keeps for the results."""
    t, m, n = _inputs(case, seed), case["rows"], case["cols"]
    state = {"case": case, "in": t, "noise": _noise(seed)}

    def new(*shape):
        return torch.empty(shape, device="cuda")

    kind = case["kind"]
    if kind in ("norm_fwd", "drop"):
        out = {"y": new(m, n)}
        if case.get("keep8"):
            state["packed"] = torch.empty(_layout(m, n)[3], dtype=torch.uint8, device="cuda")
            out["y8"] = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    elif kind == "norm_bwd":
        out = {"dx": new(m, n)} | {"d" + k: new(n) for k in ("norm_w", "norm_b") if k in t}
    elif kind == "join_fwd":
        out = {"y": new(m, n)}
        if case["next"] != "none":
            out["u"] = new(m, n)
    else:
        out = {"dx": new(m, n), "df": new(m, n)}
        if "gate" in t:
            out["dgate"] = new(case["groups"], n)
        out |= {"d" + k: new(n) for k in ("post_w", "post_b", "next_w", "next_b") if k in t}
    state["out"] = out
    return state


# ---------------------------------------------------------------- one pass, the framework's
def _context():
    global _ctx
    if _ctx is None:
        from orcaml_amd.device import Context
        _ctx = Context(0)
    return _ctx.handle


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(state):
    from orcaml_amd import _lib

    case, t, out, h = state["case"], state["in"], state["out"], _context()
    m, n, kind = case["rows"], case["cols"], case["kind"]
    seed, offset = state["noise"]
    if kind == "drop":
        _lib.call("orca_hip_dropout", h, m, n, _ptr(t["x"]), n, case["p"], seed, offset, _ptr(out["y"]), n)
        return out

    def norm(name):
        return _lib.NormParams(kind=NORMS.index(case[name]), eps=EPS, weight=_ptr(t.get(name + "_w")),
                               bias=_ptr(t.get(name + "_b")))

    if kind == "norm_fwd":
        packed = state.get("packed")
        _lib.call("orca_hip_norm", h, m, n, _ptr(t["x"]), n, ctypes.byref(norm("norm")), _ptr(out["y"]), n,
                  _ptr(packed))
        if packed is not None:  # as the values that it stands for
            _lib.call("orca_hip_act8_unpack", h, _ptr(packed), m, n, _lib.BF16, _ptr(out["y8"]), n)
        return out
    if kind == "norm_bwd":
        _lib.call("orca_hip_norm_backward", h, m, n, _ptr(t["dy"]), n, _ptr(t["x"]), n, ctypes.byref(norm("norm")),
                  _ptr(t.get("add")), n, _ptr(out["dx"]), n, _ptr(out.get("dnorm_w")), _ptr(out.get("dnorm_b")))
        return out
    s, b = _scales(case)
    block = _lib.ResidualBlock(post=norm("post"), next=norm("next"), gate=_ptr(t.get("gate")), groups=case["groups"],
                               ldgate=n, residual_scale=s, block_scale=b, p=case["p"], seed=seed, offset=offset)
    if kind == "join_fwd":
        _lib.call("orca_hip_residual_norm", h, m, n, _ptr(t["x"]), n, _ptr(t["f"]), n, ctypes.byref(block),
                  _ptr(out["y"]), n, _ptr(out.get("u")), n, None)
        return out
    grads = _lib.ResidualGrads(dx=_ptr(out["dx"]), lddx=n, df=_ptr(out["df"]), lddf=n, dgate=_ptr(out.get("dgate")),
                               lddgate=n, dpost_weight=_ptr(out.get("dpost_w")), dpost_bias=_ptr(out.get("dpost_b")),
                               dnext_weight=_ptr(out.get("dnext_w")), dnext_bias=_ptr(out.get("dnext_b")))
    _lib.call("orca_hip_residual_norm_backward", h, m, n, _ptr(t["dy"]), n, _ptr(t.get("du")), n, _ptr(t["f"]), n,
              _ptr(t["y"]), n, ctypes.byref(block), ctypes.byref(grads))
    return out


# ---------------------------------------------------------------- one pass, plain
_LOW = 0xFFFFFFFF


def _mul32(a, b):
    """The high and the low word of products of words, held in 64 bits."""
    p = a * b  # wraps, which changes no bit of either word
    return (p >> 32) & _LOW, p & _LOW


def _kept(rows, cols, p, seed, offset):
    """Which values of a matrix the dropout keeps."""
    quads = -(-cols // 4)
    c = torch.arange(rows * quads, dtype=torch.int64, device="cuda")
    c = [c % quads, c // quads, torch.full_like(c, offset & _LOW), torch.full_like(c, offset >> 32)]
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(10):
        h0, l0 = _mul32(c[0], 0xD2511F53)
        h1, l1 = _mul32(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return (torch.stack(c, 1) >= round(p * 2 ** 32)).reshape(rows, quads * 4)[:, :cols]


def _drop(v, state):
    p = state["case"]["p"]
    if p == 0:
        return v
    keep = _kept(*v.shape, p, *state["noise"])
    return torch.where(keep, v * (2 ** 32 / (2 ** 32 - round(p * 2 ** 32))), 0.0)


def _unit(kind, v):
    """The rows at mean 0 and variance 1, or at mean square 1, and 1 over their deviation."""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    r = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
    return v * r, r


def _norm(kind, t, name, v):
    if kind == "none":
        return v
    v = _unit(kind, v)[0] * t[name + "_w"]
    return v + t[name + "_b"] if name + "_b" in t else v


def _norm_grads(kind, t, name, dv, unit, r, out):
    """The gradient of the norm's input; those of its weight and bias go to `out`."""
    out["d" + name + "_w"] = (dv * unit).sum(0)
    if name + "_b" in t:
        out["d" + name + "_b"] = dv.sum(0)
    dv = dv * t[name + "_w"]
    d = dv - unit * (dv * unit).mean(1, keepdim=True)
    if kind == "layer":
        d = d - dv.mean(1, keepdim=True)
    return d * r


def _rows_of(gate, rows):
    """A gate's rows for each row."""
    return gate if gate.shape[0] in (1, rows) else gate.repeat_interleave(rows // gate.shape[0], 0)


def run(state):
    if own:
        return _own(state)
    case, t = state["case"], state["in"]
    m, n, kind = case["rows"], case["cols"], case["kind"]
    if kind == "drop":
        return {"y": _drop(t["x"], state)}
    if kind == "norm_fwd":
        y = _norm(case["norm"], t, "norm", t["x"])
        return {"y": y, "y8": _unpack(_pack(y), m, n).bfloat16()} if case["keep8"] else {"y": y}
    if kind == "norm_bwd":
        out = {"dx": None}
        dx = _norm_grads(case["norm"], t, "norm", t["dy"], *_unit(case["norm"], t["x"]), out)
        out["dx"] = dx + t["add"] if "add" in t else dx
        return out
    s, b = _scales(case)
    gate = _rows_of(t["gate"], m) if "gate" in t else None
    if kind == "join_fwd":
        v = _drop(_norm(case["post"], t, "post", t["f"]), state)
        y = t["x"] * s + (v if gate is None else v * gate) * b
        return {"y": y, "u": _norm(case["next"], t, "next", y)} if case["next"] != "none" else {"y": y}
    out, weights = {}, {}
    g = t["dy"]
    if case["next"] != "none":
        g = g + _norm_grads(case["next"], t, "next", t["du"], *_unit(case["next"], t["y"]), weights)
    dv = g * b
    if gate is not None:
        v = _drop(_norm(case["post"], t, "post", t["f"]), state)
        out["dgate"] = (dv * v).reshape(case["groups"], -1, n).sum(1)
        dv = dv * gate
    dv = _drop(dv, state)
    if case["post"] != "none":
        dv = _norm_grads(case["post"], t, "post", dv, *_unit(case["post"], t["f"]), weights)
    return {"dx": g * s, "df": dv} | out | {k: weights[k] for k in state["out"] if k in weights}


# ---------------------------------------------------------------- checkpoints
# 8-bit codes with one power-of-two step for each 32 values of a row, in one buffer: the codes [rows][cols], then
# from a multiple of 16 bytes on the step bytes [groups of 32][rows, in multiples of 16].  Step byte b stands for
# 2^(b - 133), 255 for a group that holds an infinity or a NaN.
def _layout(rows, cols):
    """(groups of 32 columns, rows in a group's row of step bytes, offset of the step bytes, bytes)."""
    groups, ld = -(-cols // 32), -(-rows // 16) * 16
    at = -(-rows * cols // 16) * 16
    return groups, ld, at, at + groups * ld


def _pack(x):
    rows, cols = x.shape
    groups, ld, at, size = _layout(rows, cols)
    wide = torch.nn.functional.pad(x, (0, groups * 32 - cols)).reshape(rows, groups, 32)
    top = (wide.view(torch.int32) & 0x7FFFFFFF).amax(2)
    byte = ((top + 0x10000) >> 23).clamp(7, 254)
    inverse = ((260 - byte) << 23).view(torch.float32)  # 2^(133 - byte)
    codes = torch.round(wide * inverse[:, :, None]).clamp(-127, 127)
    finite = top < 0x7F800000
    codes = torch.where(finite[:, :, None], codes, 0.0).to(torch.int8)
    out = torch.zeros(size, dtype=torch.uint8, device=x.device)
    out[:rows * cols] = codes.reshape(rows, groups * 32)[:, :cols].reshape(-1).view(torch.uint8)
    out[at:].view(groups, ld)[:, :rows] = torch.where(finite, byte, 255).to(torch.uint8).t()
    return out


def _unpack(packed, rows, cols):
    groups, ld, at, _ = _layout(rows, cols)
    codes = torch.nn.functional.pad(packed[:rows * cols].view(torch.int8).reshape(rows, cols).float(),
                                    (0, groups * 32 - cols)).reshape(rows, groups, 32)
    byte = packed[at:].view(groups, ld)[:, :rows].t().int()
    step = torch.where(byte == 255, float("nan"), ((byte.clamp(7, 254) - 6) << 23).view(torch.float32))
    return (codes * step[:, :, None]).reshape(rows, groups * 32)[:, :cols]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    m, n, kind = case["rows"], case["cols"], case["kind"]
    e = 4 * m * n
    if kind == "drop":
        return {"bytes": 2 * e, "flops": m * n}
    if kind == "norm_fwd":
        moved = 2 * e + 4 * n * (1 + case["bias"])
        if case["keep8"]:  # written, read back and given as values of 16 bits
            moved += 2 * _layout(m, n)[3] + 2 * m * n
        return {"bytes": moved, "flops": 7 * m * n}
    if kind == "norm_bwd":
        return {"bytes": (3 + case["add"]) * e + 4 * n * (2 + case["bias"]), "flops": 16 * m * n}
    post, nxt = case["post"] != "none", case["next"] != "none"
    params = (1 + case["bias"]) * (post + nxt)
    gate = 4 * case["groups"] * n
    if kind == "join_fwd":
        return {"bytes": (3 + nxt) * e + gate + 4 * n * params, "flops": (5 + 7 * (post + nxt)) * m * n}
    # f is read for its norm's or the gate's gradient, y and du for the next norm's
    return {"bytes": (3 + 2 * nxt + (post or case["groups"] > 0)) * e + 2 * gate + 8 * n * params,
            "flops": (6 + 16 * (post + nxt)) * m * n}


# ---------------------------------------------------------------- the same in 64 bits
def _words64(rows, cols, seed, offset):
    """The random words of a matrix [rows][cols], by products of 16-bit halves."""
    def times(m, v):
        lo, hi = (m & 65535) * v, (m >> 16) * v  # below 2^48
        low = lo + ((hi & 65535) << 16)
        return (hi >> 16) + (low >> 32), low & _LOW

    out = torch.empty((rows, -(-cols // 4), 4), dtype=torch.int64, device="cuda")
    row = torch.arange(rows, dtype=torch.int64, device="cuda")[:, None].expand(out.shape[:2])
    w, x = torch.arange(out.shape[1], dtype=torch.int64, device="cuda")[None].expand(out.shape[:2]), row
    y, z = torch.zeros_like(row) + offset % 2 ** 32, torch.zeros_like(row) + offset // 2 ** 32
    for i in range(10):
        ka = (seed % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32
        kb = (seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32
        (wh, wl), (yh, yl) = times(0xD2511F53, w), times(0xCD9E8D57, y)
        w, x, y, z = torch.bitwise_xor(yh ^ x, torch.full_like(x, ka)), yl, \
            torch.bitwise_xor(wh ^ z, torch.full_like(z, kb)), wl
    for i, v in enumerate((w, x, y, z)):
        out[:, :, i] = v
    return out.reshape(rows, -1)[:, :cols]


def _factor64(case, seed):
    """What the dropout multiplies each value with."""
    m, n, p = case["rows"], case["cols"], case["p"]
    border = round(p * 2 ** 32)
    if border == 0:
        return torch.ones((1, 1), dtype=torch.float64, device="cuda")
    return (_words64(m, n, *_noise(seed)) >= border).double() * (2.0 ** 32 / (2.0 ** 32 - border))


def _round8(v):
    """The nearest values of a checkpoint: multiples of the group's step, which is the least power of two
    that keeps every multiple within 127."""
    rows, cols = v.shape
    out = torch.empty_like(v)
    for at in range(0, cols, 32):
        part = v[:, at:at + 32]
        top = part.abs().amax(1, keepdim=True)
        mant, exp = torch.frexp(top)  # top = mant 2^exp, 0.5 <= mant < 1
        power = exp - 7 + (mant >= 127.5 / 128).int()
        power = torch.where(top > 0, power, -126).clamp(-126, 121)
        step = torch.exp2(power.double())
        out[:, at:at + 32] = torch.round(part / step).clamp(-127, 127) * step
    return out


def _stats64(kind, v):
    """(mean, 1 / deviation) of the rows."""
    mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    return mean, ((v - mean).square().mean(1, keepdim=True) + EPS).rsqrt()


def _norm64(kind, t, name, v):
    if kind == "none":
        return v
    mean, r = _stats64(kind, v)
    return (v - mean) * r * t[name + "_w"] + t.get(name + "_b", 0.0)


def _back64(kind, t, name, dv, v):
    """(gradient of v, of the weight, of the bias) of a norm."""
    mean, r = _stats64(kind, v)
    hat = (v - mean) * r
    e = dv * t[name + "_w"]
    inner = (e * hat).sum(1, keepdim=True) / v.shape[1]
    level = e.sum(1, keepdim=True) / v.shape[1] if kind == "layer" else 0.0
    return r * (e - level - hat * inner), (dv * hat).sum(0), dv.sum(0)


def exact(case, seed):
    t = {k: v.double() for k, v in _inputs(case, seed).items()}
    kind, m, n = case["kind"], case["rows"], case["cols"]
    if kind == "drop":
        return {"y": t["x"] * _factor64(case, seed)}
    if kind == "norm_fwd":
        y = _norm64(case["norm"], t, "norm", t["x"])
        return {"y": y, "y8": _round8(y)} if case["keep8"] else {"y": y}
    if kind == "norm_bwd":
        dx, dw, db = _back64(case["norm"], t, "norm", t["dy"], t["x"])
        out = {"dx": dx + t.get("add", 0.0), "dnorm_w": dw}
        return out | {"dnorm_b": db} if case["bias"] else out
    s, b = _scales(case)
    factor = _factor64(case, seed) * b
    gate = t["gate"].repeat_interleave(m // case["groups"], 0) if case["groups"] else 1.0
    v = _norm64(case["post"], t, "post", t["f"])
    if kind == "join_fwd":
        y = s * t["x"] + factor * gate * v
        return {"y": y, "u": _norm64(case["next"], t, "next", y)} if case["next"] != "none" else {"y": y}
    g, grads = t["dy"], {}
    if case["next"] != "none":
        d, grads["dnext_w"], grads["dnext_b"] = _back64(case["next"], t, "next", t["du"], t["y"])
        g = g + d
    out = {"dx": s * g}
    df = g * factor * gate
    if case["post"] != "none":
        df, grads["dpost_w"], grads["dpost_b"] = _back64(case["post"], t, "post", df, t["f"])
    out["df"] = df
    if case["groups"]:
        out["dgate"] = (g * factor * v).reshape(case["groups"], m // case["groups"], n).sum(1)
    for k in ("post_w", "post_b", "next_w", "next_b"):
        if k in t:
            out["d" + k] = grads["d" + k]
    return out
