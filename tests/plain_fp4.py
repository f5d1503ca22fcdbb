"""Microscaled 4-bit floating point from its definition, number by number in 64 bits (each 32-bit step worked out in 64 and rounded), for the tests.

Groups of 32 numbers with a power of two ("mx"), or of 16 with an 8-bit float and a factor for each row ("nv"); csrc/fp4.cuh has the formulas.
"""

import numpy as np
import torch

GROUP = {"mx": 32, "nv": 16}
FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# every finite 8-bit float with four bits of exponent and three of fraction, in order: its code is its place
E4M3 = [(m / 8) * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127]


def nearest(a, table):
    """The place of the nearest entry of ``table`` for every ``a >= 0``, ties to the even place, the last for what is above."""
    t = np.array(table)
    hi = np.clip(np.searchsorted(t, a, side="left"), 1, len(t) - 1)
    lo = hi - 1
    below, above = a - t[lo], t[hi] - a
    return np.where(below < above, lo, np.where(above < below, hi, np.where(lo % 2 == 0, lo, hi)))


def r32(a):
    with np.errstate(over="ignore", under="ignore"):
        return np.asarray(a, np.float64).astype(np.float32).astype(np.float64)


def held(x, kind):
    """(codes 0..15, scales' bytes, factors) of ``x`` [rows, k]; codes [rows, groups, group], zeros behind the row's end."""
    x = x.detach().cpu().double().numpy()
    rows, k = x.shape
    group = GROUP[kind]
    a = np.zeros((rows, -(-k // group) * group))
    a[:, :k] = x
    a = a.reshape(rows, -1, group)
    mag = np.where(np.isfinite(a), np.abs(a), 0.0)
    bad = ~np.isfinite(a).all(-1)
    top = mag.max(-1)
    if kind == "mx":
        e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2, -127)
        e = np.maximum(e, -127)
        byte, factor = e + 127, None
        y = mag / np.ldexp(1.0, e)[..., None]
    else:
        factor = np.maximum(r32(top.max(-1) / 2688.0), 2.0**-112)
        u = r32(1.0 / r32(6.0 * factor))
        byte = nearest(r32(top * u[:, None]), E4M3)
        s = np.array(E4M3)[byte]
        with np.errstate(divide="ignore"):
            r = np.where(byte > 0, r32(1.0 / r32(np.where(byte > 0, s, 1.0) * factor[:, None])), 0.0)
        y = r32(mag * r[..., None])
    c = nearest(y, FP4) + 8 * np.signbit(np.where(np.isnan(a), 0.0, a))
    c[bad] = 2
    byte = np.where(bad, 0x7F if kind == "nv" else 0xFF, byte)
    return c, byte, factor


def values(x, kind):
    """What the 4-bit form of ``x`` stands for, float64 [rows, k]."""
    c, byte, factor = held(x, kind)
    if kind == "nv":
        s = np.array(E4M3 + [np.nan])[byte]
    else:
        s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))
    v = np.array(FP4 + [-f for f in FP4])[c] * s[..., None]
    v = v.reshape(v.shape[0], -1)[:, :x.shape[1]]
    return torch.from_numpy(v if factor is None else v * factor[:, None])


def product(x, w, kind):
    """(x w^T, the sum of the terms' magnitudes), float64, from the 4-bit forms."""
    a, b = values(x, kind), values(w, kind)
    return a @ b.T, a.abs() @ b.abs().T


def silu_mul(gate_up):
    k = gate_up.shape[1] // 2
    g, u = gate_up[:, :k].double(), gate_up[:, k:].double()
    return ((g * torch.sigmoid(g)).to(gate_up.dtype).double() * u).to(gate_up.dtype)
