"""CPU oracle for the microscaled 4-bit format and the few-token layer (test infrastructure, never imported by the
product).  Everything is evaluated in 64 bits from the fields of the formats; where the quantiser's definition holds a
value in fp32, the 64-bit result is rounded to fp32 there.

E2M1: sign, two exponent bits (bias 1), one fraction bit.  E4M3: bias 7, three fraction bits, 0x7F = NaN.  E8M0:
2^(byte - 127), 0xFF = NaN (OCP Microscaling Formats, version 1.0).
"""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6])


def e4m3(b: np.ndarray) -> np.ndarray:
    b = b.astype(np.int64)
    e, f = (b >> 3) & 15, (b & 7) / 8.0
    v = np.where(e == 0, f * 2.0 ** -6, (1 + f) * 2.0 ** (e - 7.0))
    v = np.where((b & 0x7F) == 0x7F, np.nan, v)
    return np.where(b & 0x80, -v, v)


def e8m0(b: np.ndarray) -> np.ndarray:
    return np.where(b == 255, np.nan, 2.0 ** (b.astype(np.float64) - 127))


def unpack(q: np.ndarray) -> np.ndarray:
    out = np.empty((*q.shape[:-1], q.shape[-1] * 2), np.uint8)
    out[..., 0::2], out[..., 1::2] = q & 15, q >> 4
    return out


def values(q: np.ndarray, scale: np.ndarray, glob, block: int) -> np.ndarray:
    """The numbers in 64 bits; ``glob`` broadcasts over the leading dimension (None = 1)."""
    s = e4m3(scale) if block == 16 else e8m0(scale)
    v = E2M1[unpack(q)] * np.repeat(s, block, axis=-1)
    if glob is not None:
        v = v * np.asarray(glob, np.float64).reshape(-1, *([1] * (v.ndim - 1)))
    return v


def _f32(v):
    with np.errstate(over="ignore"):
        return np.asarray(v, np.float64).astype(np.float32).astype(np.float64)


def _round_to(v, lead_min, bits):
    """Nearest multiple (ties to even) of 2^(exponent - bits), the exponent at least ``lead_min``."""
    _, e = np.frexp(v)
    step = 2.0 ** (np.maximum(e - 1, lead_min) - bits)
    return np.rint(v / step) * step


def quantize(x: np.ndarray, block: int, glob: float = None):
    """One matrix [rows, cols] in 64 bits -> (codes [rows, cols], scale bytes [rows, cols/block], global)."""
    rows, cols = x.shape
    v = x.reshape(rows, cols // block, block).astype(np.float64)
    bad = ~np.isfinite(v).all(-1)
    mag = np.where(bad, 0.0, np.abs(np.where(np.isfinite(v), v, 0.0)).max(-1))
    if block == 16:
        if glob is None:
            # the computed global scale looks at every finite group of 16
            top = mag.max() if mag.size else 0.0
            glob = 1.0 if top == 0 else max(float(_f32(top / 2688.0)), 2.0 ** -110)
        with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
            t = np.minimum(_f32(mag / _f32(6.0 * glob)), 448.0)
        s = _round_to(t, -6, 3)
        unit = _f32(s * glob)
        ok = unit >= 2.0 ** -126
        s = np.where(ok, s, 0.0)
        with np.errstate(divide="ignore"):
            inv = np.where(ok, _f32(1.0 / np.where(ok, unit, 1.0)), 0.0)
        sb = np.zeros(s.shape, np.uint8)
        table = e4m3(np.arange(127, dtype=np.uint8))
        sb[...] = np.searchsorted(table, s)
        assert np.array_equal(table[sb], s)
        sb = np.where(bad, 0x7F, sb).astype(np.uint8)
    else:
        _, e = np.frexp(mag)
        e = np.where(mag > 0, np.maximum(e - 3, -127), -127)
        inv = 2.0 ** (-e.astype(np.float64))
        sb = np.where(bad, 255, e + 127).astype(np.uint8)
        ok = np.ones_like(bad)
    r = _f32(np.where(np.isfinite(v), v, 0.0) * inv[..., None])
    m = _round_to(np.minimum(np.abs(r), 6.0), 0, 1)
    idx = np.searchsorted(E2M1[:8], m)
    code = np.where(np.signbit(r), idx + 8, idx)
    code = np.where((bad | ~ok)[..., None], 0, code).astype(np.uint8)
    return code.reshape(rows, cols), sb, glob


def layer_with_bound(x, w1, w2, ids, weights, eps):
    """The layer in 64 bits for a given routing, and the largest error its rounding points allow per output element:
    the activations between the products rounded to a type with spacing ``eps`` (half a step), the products accumulated
    in fp32 in any order (n * 2^-24 of the sum of magnitudes), SiLU in fp32 through the fast exponential and division
    (documented: 2 + 1.173 |g| and 2 units in the last place), one rounding of the output."""
    x, w1, w2 = (np.asarray(a, np.float64) for a in (x, w1, w2))
    M, H = x.shape
    I = w1.shape[1] // 2
    out, err = np.zeros((M, H)), np.zeros((M, H))
    u24 = 2.0 ** -24
    for t in range(M):
        for j in range(ids.shape[1]):
            e, w = int(ids[t, j]), float(weights[t, j])
            h = w1[e] @ x[t]
            dh = (H + 8) * u24 * (np.abs(w1[e]) @ np.abs(x[t]))
            g, u, dg, du = h[:I], h[I:], dh[:I], dh[I:]
            sig = 1 / (1 + np.exp(-g))
            act = g * sig * u
            dact = 1.1 * dg * (np.abs(u) + du) + np.abs(g * sig) * du
            dact += (6 + 1.2 * np.minimum(np.abs(g), 90)) * 2.0 ** -23 * np.abs(act)
            dact = dact + eps / 2 * (np.abs(act) + dact)
            mag = np.abs(w2[e]) @ (np.abs(act) + dact)
            out[t] += w * (w2[e] @ act)
            err[t] += w * (np.abs(w2[e]) @ dact) + (I + 16 + ids.shape[1]) * u24 * w * mag
    return out, err + eps / 2 * (np.abs(out) + err)
