"""The token cache's operators in 64 bits, from their definitions: rotary positions,
e4m3 rows with a power-of-two scale, attention over packed sequences."""
import math

import numpy as np


def rope(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False):
    """x f64 [T, H, hd]; the first 2 * len(inv_freq) elements of every head turned."""
    y = np.array(x, np.float64)
    half = len(inv_freq)
    a = np.outer(np.asarray(positions, np.float64), np.asarray(inv_freq, np.float64))
    if inverse:
        a = -a
    c, s = np.cos(a)[:, None] * scale, np.sin(a)[:, None] * scale
    i0, i1 = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    x0, x1 = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def e4m3_values():
    """The 256 values of the format: 1 sign, 4 exponent (bias 7), 3 fraction bits; no
    infinities, all ones is NaN."""
    v = np.empty(256)
    for code in range(128):
        e, f = code >> 3, code & 7
        v[code] = math.nan if code == 127 else f * 2.0 ** -9 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
    v[128:] = -v[:128]
    return v


def e4m3_codes(y):
    """Codes of values in [-448, 448], nearest, ties to the even code; NaN is 0x7F or 0xFF."""
    table = e4m3_values()[:127]
    a = np.abs(y)
    hi = np.searchsorted(table, np.where(np.isnan(a), 0, a)).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    d = (table[hi] - a) - (a - table[lo])
    code = np.where((d > 0) | ((d == 0) & (lo % 2 == 0)), lo, hi)
    return (np.where(np.isnan(y), 127, code) | (np.signbit(y) << 7)).astype(np.uint8)


def quantise(x, top):
    """Rows of x (last axis) -> (codes u8, scale bytes u8).  top: the largest value that a
    rounding to four significant bits leaves finite in x's type; larger ones are held at it."""
    x = np.clip(np.asarray(x, np.float64), -top, top)
    amax = np.nanmax(np.where(np.isnan(x), 0, np.abs(x)), -1)
    m, e = np.frexp(amax / 448)                # amax / 448 = m 2^e, m in [0.5, 1)
    byte = np.maximum(1, np.where(amax > 0, e - (m == 0.5) + 127, 1))
    return e4m3_codes(x * 2.0 ** (127.0 - byte)[..., None]), byte.astype(np.uint8)


def values(codes, byte):
    return e4m3_values()[codes] * 2.0 ** (byte.astype(np.float64) - 127)[..., None]


def attention(q, k, v, causal=True, scale=None):
    """One sequence, f64: q [n, H, hd], k, v [m, Hkv, hd] -> (out [n, H, hd], the same with
    |v| for v, the largest sum of |products| of a score).  Rows that see no key are zero;
    what a row does not see does not reach it."""
    n, H, hd = q.shape
    m, Hkv = k.shape[:2]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out, mag, most = np.zeros_like(q), np.zeros_like(q), 0.0
    for h in range(H):
        g = h // (H // Hkv)
        with np.errstate(invalid='ignore'):
            s = q[:, h] @ k[:, g].T * scale
        see = np.arange(m)[None] <= np.arange(n)[:, None] + (m - n if causal else m)
        s = np.where(see, s, -np.inf)
        if m:
            b = (np.abs(q[:, h]) @ np.abs(k[:, g]).T * scale)[see]
            most = max(most, float(np.max(b[np.isfinite(b)], initial=0.0)))
            top = s.max(-1, keepdims=True)
            with np.errstate(invalid='ignore'):
                p = np.exp(s - np.where(np.isneginf(top), 0.0, top))
            l = p.sum(-1)
            bad = ~np.isfinite(v[:, g])
            vz = np.where(bad, 0.0, v[:, g])
            with np.errstate(invalid='ignore', divide='ignore'):
                o, a = p @ vz / l[:, None], p @ np.abs(vz) / l[:, None]
            o[l == 0], a[l == 0] = 0.0, 0.0
            for j in np.nonzero(bad.any(-1))[0]:
                with np.errstate(invalid='ignore'):
                    o[see[:, j]] += np.where(bad[j], v[j, g], 0.0)
            out[:, h], mag[:, h] = o, a
    return out, mag, most
