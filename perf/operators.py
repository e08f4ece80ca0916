"""The layer of a residual feed-forward block and its 8-bit activation checkpoints, as measurable cases.

  fwd    y = act(x W + b) + r in one call; it may keep the pre-activation z, or 8-bit checkpoints of z and y
  bwd    dx (with the gradient that came past the layer added), dW and db from dy and what the forward
         kept: x and z themselves or their checkpoints
  pack   an activation matrix to its checkpoint and back

A checkpoint holds a matrix as 8-bit codes with one power-of-two step for each 32 values of a row, in one
buffer: the codes [rows][cols], then from a multiple of 16 bytes on the step bytes [groups of 32][rows, in
multiples of 16].  Step byte b stands for 2^(b - 133), 255 for a group that holds an infinity or a NaN.
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # one sample through a wide layer, as an evaluation loop or a service asks for it: latency, and the weights
        {"name": "fwd_one_row", "kind": "fwd", "rows": 1, "in": 4096, "out": 4096, "act": "gelu", "residual": True,
         "keep": "none"},
        # the first layer of the smallest configuration of the repository
        {"name": "fwd_small", "kind": "fwd", "rows": 64, "in": 784, "out": 128, "act": "relu", "residual": False,
         "keep": "none"},
        # odd widths and the last, partial batch of an epoch, training (z kept)
        {"name": "fwd_ragged", "kind": "fwd", "rows": 777, "in": 1003, "out": 1501, "act": "silu", "residual": True,
         "keep": "z"},
        # the hidden layer of the benchmark's configuration, training
        {"name": "fwd_hidden", "kind": "fwd", "rows": 1024, "in": 4096, "out": 4096, "act": "gelu_tanh",
         "residual": True, "keep": "z"},
        # a large batch whose activations are kept in 8 bits
        {"name": "fwd_large_8bit", "kind": "fwd", "rows": 8192, "in": 4096, "out": 4096, "act": "gelu",
         "residual": True, "keep": "8bit"},
        # the backward of the smallest configuration's hidden layer: launches
        {"name": "bwd_small", "kind": "bwd", "rows": 64, "in": 128, "out": 128, "act": "relu", "residual": False,
         "keep": "z"},
        # the middle configuration's hidden layer
        {"name": "bwd_medium", "kind": "bwd", "rows": 256, "in": 1024, "out": 1024, "act": "gelu", "residual": True,
         "keep": "z"},
        # odd widths, from checkpoints
        {"name": "bwd_ragged_8bit", "kind": "bwd", "rows": 777, "in": 1003, "out": 1501, "act": "silu",
         "residual": False, "keep": "8bit"},
        # a layer that fills the GPU, from what the forward kept in 32 bits
        {"name": "bwd_large", "kind": "bwd", "rows": 4096, "in": 4096, "out": 4096, "act": "gelu", "residual": True,
         "keep": "z"},
        # the large batch again, from checkpoints
        {"name": "bwd_large_8bit", "kind": "bwd", "rows": 8192, "in": 4096, "out": 4096, "act": "gelu",
         "residual": True, "keep": "8bit"},
        # a small activation: launches
        {"name": "pack_small", "kind": "pack", "rows": 64, "cols": 1000},
        # the activation of a large batch: memory
        {"name": "pack_large", "kind": "pack", "rows": 8192, "cols": 4096},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, spread over the logarithm; about half are multiples of 8."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 8:
        n = n // 8 * 8
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(["fwd", "fwd", "fwd", "bwd", "bwd", "bwd", "pack"])
    if kind == "pack":
        return {"kind": kind, "rows": _size(rng, 1, 8192), "cols": _size(rng, 8, 4096)}
    return {"kind": kind, "rows": _size(rng, 1, 8192), "in": _size(rng, 16, 4096), "out": _size(rng, 16, 4096),
            "act": rng.choice(ACTS), "residual": rng.random() < 0.5,
            "keep": rng.choice(["none", "z", "8bit"] if kind == "fwd" else ["z", "8bit"])}


# ---------------------------------------------------------------- checkpoints
def _layout(rows, cols):
    """(groups of 32 columns, rows in a group's row of step bytes, offset of the step bytes, bytes)."""
    groups, ld = -(-cols // 32), -(-rows // 16) * 16
    at = -(-rows * cols // 16) * 16
    return groups, ld, at, at + groups * ld


def _pack(x):
    """The checkpoint of x [rows][cols] as a buffer of bytes."""
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
    """What a checkpoint stands for, in 32 bits."""
    groups, ld, at, _ = _layout(rows, cols)
    codes = torch.nn.functional.pad(packed[:rows * cols].view(torch.int8).reshape(rows, cols).float(),
                                    (0, groups * 32 - cols)).reshape(rows, groups, 32)
    byte = packed[at:].view(groups, ld)[:, :rows].t().int()
    step = torch.where(byte == 255, float("nan"), ((byte.clamp(7, 254) - 6) << 23).view(torch.float32))
    return (codes * step[:, :, None]).reshape(rows, groups * 32)[:, :cols]


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _features(g, shape):
    """Activations: features of unequal size."""
    return _normal(g, shape) * torch.exp(_normal(g, (1, shape[1]), 0.5))


def _inputs(case, seed):
    """A layer inside a network: weights of a model under training, the batch's activations and, for the
    backward, the gradient of a mean loss and what the forward kept."""
    g = _gen(seed)
    if case["kind"] == "pack":
        return {"x": _features(g, (case["rows"], case["cols"]))}
    m, k, n = case["rows"], case["in"], case["out"]
    t = {"x": _features(g, (m, k)), "w": (torch.rand((k, n), generator=g, device="cuda") * 2 - 1) / math.sqrt(k),
         "b": _normal(g, (n,), 0.1)}
    if case["kind"] == "fwd":
        if case["residual"]:
            t["r"] = _features(g, (m, n))
        return t
    t["dy"] = _normal(g, (m, n), 1.0 / m)
    if case["residual"]:
        t["add"] = _normal(g, (m, k), 1.0 / m)
    z = t["x"] @ t["w"] + t["b"]
    if case["keep"] == "8bit":
        t["x8"], t["z8"] = _pack(t.pop("x")), _pack(z)
    else:
        t["z"] = z
    return t


_ctx = None


def prepare(case, seed):
    """The inputs, and the buffers that a program keeps for the results."""
    t = _inputs(case, seed)
    state = {"case": case, "in": t}
    if case["kind"] == "pack":
        m, n = case["rows"], case["cols"]
        state["packed"] = torch.empty(_layout(m, n)[3], dtype=torch.uint8, device="cuda")
        state["out"] = {"x": torch.empty((m, n), device="cuda")}
        return state
    m, k, n = case["rows"], case["in"], case["out"]
    if case["kind"] == "bwd":
        state["out"] = {"dx": torch.empty((m, k), device="cuda"), "dw": torch.empty((k, n), device="cuda"),
                        "db": torch.empty(n, device="cuda")}
        return state
    out = {"y": torch.empty((m, n), device="cuda")}
    if case["keep"] == "z":
        out["z"] = torch.empty((m, n), device="cuda")
    if case["keep"] == "8bit":
        state["packed"] = [torch.empty(_layout(m, n)[3], dtype=torch.uint8, device="cuda") for _ in range(2)]
        out |= {k: torch.empty((m, n), dtype=torch.bfloat16, device="cuda") for k in ("z8", "y8")}
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
    if case["kind"] == "pack":
        m, n = case["rows"], case["cols"]
        _lib.call("orca_hip_act8_pack", h, _ptr(t["x"]), m, n, n, _ptr(state["packed"]))
        _lib.call("orca_hip_act8_unpack", h, _ptr(state["packed"]), m, n, _lib.F32, _ptr(out["x"]), n)
        return out
    m, k, n, act = case["rows"], case["in"], case["out"], ACTS.index(case["act"])
    if case["kind"] == "fwd":
        z8, y8 = state.get("packed", (None, None))
        epi = _lib.LinearEpilogue(act=act, bias=_ptr(t["b"]), residual=_ptr(t.get("r")), ldr=n, pre=_ptr(out.get("z")),
                                  ldpre=n, pre8=_ptr(z8), y8=_ptr(y8))
        _lib.call("orca_hip_linear_act", h, m, n, k, _ptr(t["x"]), k, _ptr(t["w"]), n, _ptr(out["y"]), n,
                  ctypes.byref(epi))
        if z8 is not None:  # as the values that they stand for
            _lib.call("orca_hip_act8_unpack", h, _ptr(z8), m, n, _lib.BF16, _ptr(out["z8"]), n)
            _lib.call("orca_hip_act8_unpack", h, _ptr(y8), m, n, _lib.BF16, _ptr(out["y8"]), n)
        return out
    saved = _lib.LinearSaved(act=act, z=_ptr(t.get("z")), ldz=n, z8=_ptr(t.get("z8")), x=_ptr(t.get("x")), ldx=k,
                             x8=_ptr(t.get("x8")), dx_add=_ptr(t.get("add")), ldadd=k)
    _lib.call("orca_hip_linear_act_backward", h, m, n, k, _ptr(t["dy"]), n, _ptr(t["w"]), n, ctypes.byref(saved),
              _ptr(out["dx"]), k, _ptr(out["dw"]), n, _ptr(out["db"]))
    return out


# ---------------------------------------------------------------- one pass, plain
_C, _A = math.sqrt(2 / math.pi), 0.044715


def _act(kind, z):
    if kind == "relu":
        return torch.where(z > 0, z, 0.0)
    if kind == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return z / (1 + torch.exp(-2 * _C * (z + _A * z * z * z)))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(kind, z):
    if kind == "relu":
        return (z > 0).float()
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        s = 1 / (1 + torch.exp(-2 * _C * (z + _A * z * z * z)))
        return s + z * s * (1 - s) * (2 * _C) * (1 + 3 * _A * z * z)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def run(state):
    if own:
        return _own(state)
    case, t = state["case"], state["in"]
    if case["kind"] == "pack":
        return {"x": _unpack(_pack(t["x"]), case["rows"], case["cols"])}
    m, k, n = case["rows"], case["in"], case["out"]
    if case["kind"] == "fwd":
        z = t["x"] @ t["w"] + t["b"]
        y = _act(case["act"], z)
        if "r" in t:
            y = y + t["r"]
        out = {"y": y}
        if case["keep"] == "z":
            out["z"] = z
        if case["keep"] == "8bit":
            out["z8"], out["y8"] = (_unpack(_pack(v), m, n).bfloat16() for v in (z, y))
        return out
    x, z = (_unpack(t["x8"], m, k), _unpack(t["z8"], m, n)) if "x8" in t else (t["x"], t["z"])
    dz = t["dy"] if case["act"] == "none" else t["dy"] * _slope(case["act"], z)
    dx = dz @ t["w"].t()
    if "add" in t:
        dx = dx + t["add"]
    return {"dx": dx, "dw": x.t() @ dz, "db": dz.sum(0)}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "pack":
        n, p = case["rows"] * case["cols"], _layout(case["rows"], case["cols"])[3]
        return {"bytes": 8 * n + 2 * p, "flops": 4 * n}
    m, k, n = case["rows"], case["in"], case["out"]
    if case["kind"] == "fwd":
        moved = 4 * (m * k + k * n + n + m * n) + 4 * m * n * case["residual"] + 4 * m * n * (case["keep"] == "z")
        if case["keep"] == "8bit":  # written, read back and given as values of 16 bits
            moved += 2 * (2 * _layout(m, n)[3] + 2 * m * n)
        return {"bytes": moved, "flops": 2 * m * k * n}
    kept = _layout(m, k)[3] + _layout(m, n)[3] if case["keep"] == "8bit" else 4 * m * (k + n)
    return {"bytes": 4 * (m * n + 2 * k * n + m * k + n) + kept + 4 * m * k * case["residual"],
            "flops": 4 * m * k * n}


# ---------------------------------------------------------------- the same in 64 bits
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


def _act64(kind, z):
    """(act(z), its derivative)."""
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        th = torch.tanh(_C * (z + _A * z ** 3))
        return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th ** 2) * _C * (1 + 3 * _A * z ** 2)
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    return z, torch.ones_like(z)


def _read64(packed, rows, cols):
    groups, ld, at, _ = _layout(rows, cols)
    power = packed[at:].view(groups, ld)[:, :rows].t().double() - 133
    return packed[:rows * cols].view(torch.int8).view(rows, cols).double() \
        * torch.exp2(power).repeat_interleave(32, 1)[:, :cols]


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "pack":
        return {"x": _round8(t["x"].double())}
    m, k, n = case["rows"], case["in"], case["out"]
    w = t["w"].double()
    if case["kind"] == "fwd":
        z = t["x"].double() @ w + t["b"].double()
        y = _act64(case["act"], z)[0]
        if "r" in t:
            y = y + t["r"].double()
        out = {"y": y}
        if case["keep"] == "z":
            out["z"] = z
        if case["keep"] == "8bit":
            out |= {"z8": _round8(z), "y8": _round8(y)}
        return out
    x, z = (_read64(t["x8"], m, k), _read64(t["z8"], m, n)) if "x8" in t else (t["x"].double(), t["z"].double())
    dz = t["dy"].double() * _act64(case["act"], z)[1]
    dx = dz @ w.t()
    if "add" in t:
        dx = dx + t["add"].double()
    return {"dx": dx, "dw": x.t() @ dz, "db": dz.sum(0)}
