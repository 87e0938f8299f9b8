"""The four-bit block products and the norms around a residual block, in float64 numpy.

Oracle for the operators of include/afir_hip_kernels.h that have no counterpart in the reference; test
infrastructure, written from the formulas in that header and from the MX format's definition (32 numbers share a
power of two, elements are e2m1).
"""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
MIDPOINTS = (GRID[1:] + GRID[:-1]) / 2


def quantize(x):
    """x [R, K] (any float dtype, exact in float64) -> codes uint8 [R, Kb*16], scale bytes uint8 [R, Kb], values
    float64 [R, K].  A number is placed among the midpoints of the grid; a midpoint goes to the even code."""
    x = np.asarray(x, dtype=np.float64)
    r, k = x.shape
    kb = -(-k // 32)
    full = np.zeros((r, kb * 32))
    full[:, :k] = x
    full = full.reshape(r, kb, 32)
    bad = ~np.isfinite(full).all(axis=2)
    clean = np.where(bad[:, :, None], 0.0, full)
    top = np.abs(clean).max(axis=2) if k else np.zeros((r, kb))
    exponent = np.full(top.shape, -127)
    some = top > 0
    exponent[some] = np.maximum(np.frexp(top[some])[1] - 3, -127)
    z = np.abs(clean) * np.exp2(-exponent.astype(np.float64))[:, :, None]
    below = np.searchsorted(MIDPOINTS, z, side="left")      # midpoints strictly under z
    upto = np.searchsorted(MIDPOINTS, z, side="right")      # ... or equal to it
    code = np.where(below == upto, below, np.where(below % 2 == 0, below, upto)).astype(np.uint8)
    values = GRID[code] * np.exp2(exponent.astype(np.float64))[:, :, None]
    values = np.where(np.signbit(clean), -values, values)
    code = code + np.where(np.signbit(full) & ~bad[:, :, None], 8, 0).astype(np.uint8)
    values = np.where(bad[:, :, None], np.nan, values).reshape(r, kb * 32)[:, :k]
    flat = code.reshape(r, kb * 32)
    scales = np.where(bad, 255, exponent + 127).astype(np.uint8)
    return (flat[:, 0::2] | (flat[:, 1::2] << 4)).astype(np.uint8), scales, values


def decode(codes, scales):
    """The numbers that codes [R, Kb*16] and scale bytes [R, Kb] stand for, float64 [R, Kb*32]."""
    r, kb = scales.shape
    nibbles = np.stack([codes & 15, codes >> 4], axis=2).reshape(r, kb, 32)
    v = np.where(nibbles & 8, -GRID[nibbles & 7], GRID[nibbles & 7])
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[:, :, None]).reshape(r, kb * 32)


def matmul(a, b, bias, alpha):
    """max(v, v * alpha), v = a @ b.T + bias, and the sum of the terms' magnitudes."""
    v = a @ b.T
    size = np.abs(a) @ np.abs(b).T
    if bias is not None:
        v, size = v + bias, size + np.abs(bias)
    return np.maximum(v, v * alpha), size


def rstd(v, eps):
    return 1.0 / np.sqrt((v * v).mean(axis=1, keepdims=True) + eps)


def gate_of_rows(gate, m, rows_per_gate):
    return 1.0 if gate is None else gate[np.arange(m) // rows_per_gate]


def norm(x, f, post, gate, pre, scale, eps, rows_per_gate):
    """(y, h); f, gate, pre may be None."""
    y = x if f is None else scale * x + gate_of_rows(gate, len(x), rows_per_gate) * (f * rstd(f, eps)) * post
    return y, None if pre is None else y * rstd(y, eps) * pre


def norm_grad(dy, dh, y, f, post, gate, pre, scale, eps, rows_per_gate):
    """The gradients, and for each the sum of the magnitudes that it is made of (what a rounding error is relative to)."""
    m = len(y)
    g = gate_of_rows(gate, m, rows_per_gate)
    out, size = {}, {}
    t = np.zeros_like(y) if dy is None else dy.copy()
    st = np.abs(t)
    if dh is not None:
        ry = rstd(y, eps)
        yn, a = y * ry, dh * pre
        t = t + ry * (a - yn * (a * yn).mean(axis=1, keepdims=True))
        st = st + ry * (np.abs(a) + np.abs(yn) * np.abs(a * yn).mean(axis=1, keepdims=True))
        out["dpre_weight"], size["dpre_weight"] = (dh * yn).sum(axis=0), np.abs(dh * yn).sum(axis=0)
    out["dx"], size["dx"] = scale * t, abs(scale) * st
    if f is not None:
        rf = rstd(f, eps)
        fn, b, sb = f * rf, t * g * post, st * np.abs(g * post)
        out["df"] = rf * (b - fn * (b * fn).mean(axis=1, keepdims=True))
        size["df"] = rf * (sb + np.abs(fn) * (sb * np.abs(fn)).mean(axis=1, keepdims=True))
        out["dpost_weight"], size["dpost_weight"] = (t * g * fn).sum(axis=0), (st * np.abs(g * fn)).sum(axis=0)
        if gate is not None:
            starts = np.arange(0, m, rows_per_gate)
            out["dgate"] = np.add.reduceat(t * fn * post, starts, axis=0)
            size["dgate"] = np.add.reduceat(st * np.abs(fn * post), starts, axis=0)
    return out, size
