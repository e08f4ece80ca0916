"""Norms of rows, dropout and the joint of two residual blocks in 64 bits, with bounds on what fp32 may be off by.

U = 2^-24 is half a step of fp32, relative.  A sum of n terms that runs over `s` additions at most for each term is off
by at most s U times the sum of magnitudes (to first order in U; the bounds below leave out terms in U^2).  A row's sums
run over at most steps(n) additions: a thread adds up to n / 64 values if that is at most 16, else n / 256 (rows are
held by 64 threads up to 1024 values, by 256 and more above), then 6 additions over a wave, 3 over a block's
waves (up to 7 where a row takes 8 waves) and the sum of four neighbours."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24


def steps(n):
    return max(min(n / 64, 16), n / 256) + 16


# ---------------------------------------------------------------- Philox4x32-10
def philox(counter, key):
    """The four words of 32 bits for a counter of four and a key of two, each an array or a number."""
    c = [np.asarray(v, np.uint64) for v in counter]
    k = [int(v) for v in key]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]),
             a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def dropout_factor(rows, cols, p, seed, offset):
    """What a dropout multiplies each value with: 0, or one over the share of words that keep."""
    border = round(p * 2 ** 32)
    if border == 0:
        return np.ones((rows, cols))
    quads = -(-cols // 4)
    q = np.broadcast_to(np.arange(quads, dtype=np.uint64)[None], (rows, quads))
    r = np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], (rows, quads))
    zero = np.zeros((rows, quads), np.uint64)
    w = philox([q, r, zero + np.uint64(offset % 2 ** 32), zero + np.uint64(offset >> 32)],
               [seed % 2 ** 32, seed >> 32])
    keep = np.stack(w, 2).reshape(rows, 4 * quads)[:, :cols] >= border
    return keep * (2.0 ** 32 / (2.0 ** 32 - border) if border < 2 ** 32 else 0.0)


# ---------------------------------------------------------------- norms
def unit(kind, v, eps, tv=0.0, rounded_mean=False):
    """(unit(v), r, bound on unit's error) for rows v known to tv.  In fp32 a difference to the mean is off by U of
    itself; the mean is corrected by the sum of the differences, so it is off by (steps + 1) U of their mean
    magnitude, which is at most the deviation, or 1 in units of it; where it is then rounded to one fp32 value, by U of
    itself more.  The mean square is off by (steps + 3) U of itself, r by half that and three roundings."""
    n = v.shape[1]
    mean = v.mean(1, keepdims=True) if kind == "layer" else np.zeros((v.shape[0], 1))
    r = 1 / np.sqrt(((v - mean) ** 2).mean(1, keepdims=True) + np.float64(np.float32(eps)))
    u = (v - mean) * r
    tol = U * (np.abs(u) * ((steps(n) + 3) / 2 + 6) + (kind == "layer") * (steps(n) + 3))
    if rounded_mean:
        tol = tol + U * np.abs(mean) * r
    tv = np.broadcast_to(tv, v.shape)
    # a change of v by tv moves the mean by its mean and r by at most r mean(|unit| tv) r
    tol = tol + r * (tv + (kind == "layer") * tv.mean(1, keepdims=True)
                     + np.abs(u) * (np.abs(u) * tv).mean(1, keepdims=True))
    return u, r, tol


def norm(kind, v, eps, w, b, tv=0.0, rounded_mean=False):
    """(norm(v), bound)."""
    if kind == "none":
        return v, np.broadcast_to(tv, v.shape)
    u, _, tol = unit(kind, v, eps, tv, rounded_mean)
    return u * w + b, np.abs(w) * tol + 2 * U * (np.abs(u * w) + np.abs(b))


def sums(terms, tterms):
    """Column sums and their bound; rows are added one after the other at most."""
    return terms.sum(0), tterms.sum(0) + U * (terms.shape[0] + 2) * np.abs(terms).sum(0)


def norm_back(kind, v, eps, w, dv, tdv=0.0):
    """((dv of the input, bound), (dw, bound), (db, bound)) for a gradient dv known to tdv."""
    n = v.shape[1]
    u, r, tu = unit(kind, v, eps, rounded_mean=True)
    tdv = np.broadcast_to(tdv, dv.shape)
    e, te = dv * w, np.abs(w) * tdv + U * np.abs(dv * w)
    s = U * (steps(n) + 2)
    c1 = e.mean(1, keepdims=True) if kind == "layer" else np.zeros_like(r)
    t1 = s * np.abs(e).mean(1, keepdims=True) + te.mean(1, keepdims=True) if kind == "layer" else np.zeros_like(r)
    c2 = (e * u).mean(1, keepdims=True)
    t2 = (s * np.abs(e * u) + te * np.abs(u) + np.abs(e) * tu).mean(1, keepdims=True)
    d = e - c1 - u * c2
    # r is off by (steps + 3) / 2 + 3 roundings, the expression by four of its largest parts
    td = te + t1 + np.abs(u) * t2 + tu * np.abs(c2) + 4 * U * (np.abs(e) + np.abs(c1) + np.abs(u * c2))
    td = td + U * ((steps(n) + 3) / 2 + 4) * np.abs(d)
    return (d * r, td * r), sums(dv * u, tdv * np.abs(u) + np.abs(dv) * tu), sums(dv, tdv)


# ---------------------------------------------------------------- the joint
def gate_rows(gate, rows):
    return np.repeat(gate, rows // gate.shape[0], 0) if gate is not None else np.ones((1, 1))


def joint(x, f, b):
    """{"y": (value, bound), "u": ...} for parameters b: post, next = (kind, eps, w, b), gate, rs, bs, factor."""
    v, tv = norm(b["post"][0], f, *b["post"][1:])
    k = b["bs"] * b["factor"] * gate_rows(b["gate"], x.shape[0])
    # k is off by two roundings and the scale's, its product and the sum with x by one each
    t = k * v
    with np.errstate(invalid="ignore"):
        y, ty = b["rs"] * x + t, np.abs(k) * tv + 5 * U * np.abs(t) + 2 * U * (np.abs(b["rs"] * x) + np.abs(t))
    out = {"y": (y, ty)}
    if b["next"][0] != "none":
        out["u"] = norm(b["next"][0], y, *b["next"][1:], tv=ty)
    return out


def joint_back(dy, du, f, y, b):
    """{"dx", "df", "dgate", "dpost_weight", ...: (value, bound)}."""
    out = {}
    g = np.zeros(f.shape) if dy is None else dy
    tg = np.zeros(f.shape)
    if du is not None:
        (d, tg), out["dnext_weight"], out["dnext_bias"] = norm_back(*_nvewdv(b["next"], y, du))
        g = g + d
        tg = tg + 2 * U * (np.abs(d) + (0.0 if dy is None else np.abs(dy)))
    out["dx"] = b["rs"] * g, abs(b["rs"]) * tg + 2 * U * np.abs(b["rs"] * g)
    k = b["bs"] * b["factor"]
    dv, tdv = g * k, np.abs(k) * tg + 4 * U * np.abs(g * k)
    gate = b["gate"]
    if gate is not None:
        v, tv = norm(b["post"][0], f, *b["post"][1:], rounded_mean=True)
        each = dv * v
        teach = tdv * np.abs(v) + np.abs(dv) * tv + 2 * U * np.abs(each)
        parts = [sums(each[i:i + f.shape[0] // gate.shape[0]], teach[i:i + f.shape[0] // gate.shape[0]])
                 for i in range(0, f.shape[0], f.shape[0] // gate.shape[0])]
        out["dgate"] = np.stack([p[0] for p in parts]), np.stack([p[1] for p in parts])
        rows = gate_rows(gate, f.shape[0])
        dv, tdv = dv * rows, tdv * np.abs(rows) + U * np.abs(dv * rows)
    if b["post"][0] != "none":
        (dv, tdv), out["dpost_weight"], out["dpost_bias"] = norm_back(*_nvewdv(b["post"], f, dv), tdv=tdv)
    out["df"] = dv, tdv
    return out


def _nvewdv(n, v, dv):
    return n[0], v, n[1], n[2], dv
