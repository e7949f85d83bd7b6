"""The microscaled formats in 64 bits, from their definition: a table of the format's values and
a search for the nearest."""
import numpy as np

BLOCK = 32
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
# code 0..126: subnormals m / 8 * 2^-6, then (1 + m / 8) * 2^(e - 7); code 127 is NaN
E4M3 = np.array([(c & 7) / 8 * 2.0 ** -6 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7)
                 for c in range(127)])


def grid(fmt):
    return E4M3 if fmt == "fp8" else E2M1


def scale_bytes(amax, fmt):
    """The smallest s >= -127 with amax <= 464 * 2^s (fp8) or amax < 7 * 2^s (fp4), plus 127."""
    amax = np.asarray(amax, np.float64)
    out = np.full(amax.shape, 255, np.int64)
    for s in range(127, -128, -1):  # ends with the smallest that fits
        with np.errstate(over="ignore"):
            fits = amax <= 464 * 2.0 ** s if fmt == "fp8" else amax < 7 * 2.0 ** s
        out = np.where(fits, s + 127, out)
    return np.where(np.isfinite(amax), out, 255).astype(np.uint8)


def quantize(v, fmt):
    """codes, scales (uint8) of float64 rows."""
    v = np.asarray(v, np.float64)
    rows, cols = v.shape
    b = v.reshape(rows, cols // BLOCK, BLOCK)
    amax = np.where(np.isfinite(b).all(-1), np.abs(b).max(-1), np.inf)
    sc = scale_bytes(amax, fmt)
    bad = sc == 255
    a = np.where(bad[..., None], 0, np.abs(b)) / 2.0 ** (np.where(bad, 127, sc)[..., None].astype(np.float64) - 127)
    g = grid(fmt)
    hi = np.clip(np.searchsorted(g, a), 1, len(g) - 1)
    lo = hi - 1
    dl, dh = a - g[lo], g[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    sign = np.signbit(b) & ~bad[..., None]
    code = (code + sign * (128 if fmt == "fp8" else 8)).astype(np.uint8).reshape(rows, cols)
    if fmt == "fp4":
        code = code[:, 0::2] | (code[:, 1::2] << 4)
    return code, sc


def values(codes, scales, fmt):
    """What codes and scales stand for, in float64 (NaN where the scale is 255)."""
    if fmt == "fp4":
        codes = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
        v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    else:
        v = np.append(E4M3, np.nan)[codes & 127] * np.where(codes & 128, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * np.repeat(s, BLOCK, axis=1)


def bf16_round(v):
    """float64 -> bf16 bits, to nearest even, once (finite values and infinities)."""
    v = np.asarray(v, np.float64)
    with np.errstate(over="ignore"):
        f = v.astype(np.float32)  # then settle the double rounding: round to odd first
    bits = f.view(np.uint32).astype(np.int64)
    exact = f.astype(np.float64) == v
    away = np.abs(f.astype(np.float64)) > np.abs(v)
    trunc = np.where(~exact & away, bits - 1, bits)
    odd = np.where(~exact, trunc | 1, trunc)
    r = (odd + 0x7FFF + ((odd >> 16) & 1)) >> 16
    return np.where(np.isnan(v), 0x7FC0, r).astype(np.uint16)
