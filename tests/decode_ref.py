"""The 4-bit product, the norms on both sides and the token draw in 64 bits, from their formulas."""
import math

import numpy as np

RANGE = 28.0


def bf16_values(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def to_bf16_bits(v):
    """float32 -> bf16 bits of inputs (nearest, ties to even; finite or infinite)."""
    b = np.asarray(v, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


# ---------------------------------------------------------------- 4-bit product
def pack(q):
    """Codes 0..15 [.., K] -> bytes [.., K / 2], the even column low."""
    q = q.astype(np.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4)


def w4_product(x, q, scales, zeros, group):
    """x [N, K], q [M, K], scales [M, K / g], zeros of that shape or None; also the sum of magnitudes
    that the operator's fp32 sums go over: |x| (16 + q + 16 + z) s."""
    z = np.full(scales.shape, 8.0) if zeros is None else zeros.astype(np.float64)
    rep = lambda a: np.repeat(a.astype(np.float64), group, axis=1)  # noqa: E731
    s = rep(scales)
    with np.errstate(invalid="ignore"):
        y = x.astype(np.float64) @ ((q - rep(z)) * s).T
        mag = np.abs(x.astype(np.float64)) @ ((32 + q + rep(z)) * np.abs(s)).T
    return y, mag


def w4_bound(mag, k, group, value, f32):
    """How far an output may be off: a product is exact; it passes at most 2 group additions in its
    group's chain (64 within the instructions' order, which is not fixed), one for the scale and one
    for each group and each of up to 16 waves, each off by less than 2^-23 of the magnitudes' sum;
    then half a step of the output's type (bf16 2^-8, and below the smallest normal half a step of
    it)."""
    n = 2 * group + k // group + 18
    out = np.abs(value) * (2.0 ** -24 if f32 else 2.0 ** -8) + 2.0 ** -134
    return n * 2.0 ** -23 * mag * (1 if f32 else 1 + 2.0 ** -8) + out


# ---------------------------------------------------------------- norms on both sides
def sandwich(x, residual, pre, eps, post=None, gate=None, scale=1.0, offset=False):
    """s and z; x, residual [rows, cols], gate broadcastable."""
    one = 1.0 if offset else 0.0
    y = x.astype(np.float64)
    if post is not None:
        y = y / np.sqrt((y * y).mean(1, keepdims=True) + eps) * (one + post.astype(np.float64))
    if gate is not None:
        y = y * gate.astype(np.float64)
    s = y if residual is None else scale * residual.astype(np.float64) + y
    if pre is None:
        return s, None
    return s, s / np.sqrt((s * s).mean(1, keepdims=True) + eps) * (one + pre.astype(np.float64))


def assert_rounded(bits, v, what=""):
    """bf16 bits are v rounded to nearest, where v is known to 2^-40 of itself."""
    got = bf16_values(bits).astype(np.float64)
    exp = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -126)))
    half = 2.0 ** (exp - 8)
    bad = ~(np.abs(got - v) <= half + 2.0 ** -40 * np.abs(v))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}"


# ---------------------------------------------------------------- token draw
def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """token, logprob of one row (float32 logits)."""
    l = np.asarray(logits, np.float64).copy()
    l[np.isnan(l)] = -np.inf
    top = l.max()
    if top == -np.inf:
        return -1, -np.inf
    if top == np.inf:
        d = np.where(l == np.inf, 0.0, -np.inf)
    else:
        d = l - top
    t = float(temperature)
    if not t > 0:
        t, top_k = 1.0, 1
    t = min(t, float(np.finfo(np.float32).max))
    least = -RANGE * t
    if min_p > 0:
        least = max(least, t * math.log(min(float(min_p), 1.0)))
    live = np.flatnonzero((d >= least) & (d > -np.inf))
    order = live[np.argsort(-l[live], kind="stable")]
    if top_k > 0:
        order = order[:top_k]
    w = np.exp(d[order] / t)
    if top_p < 1:
        before = np.cumsum(w) - w
        keep = before < max(float(top_p), 0.0) * w.sum()
        keep[0] = True
        order, w = order[keep], w[keep]
    at = np.argsort(order)
    order, w = order[at], w[at]
    cum = np.cumsum(w)
    u = float(u)
    if not u > 0:
        u = 0.0
    i = min(int((cum <= u * cum[-1]).sum()), len(order) - 1)
    return int(order[i]), float(np.log(w[i] / cum[-1]))
