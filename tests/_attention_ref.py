"""Plain NumPy forms, in 64 bits, of the head norm and rotation, the MX cache coding and the
attention over it: what the tests of those operators compare with."""

import numpy as np

import mxfp4_ref as oracle

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
E2M1_BOTH = np.concatenate([E2M1, -E2M1])


def norm_rope(x, cos, sin, weight, eps, interleaved):
    """x [tokens, heads, dim]; cos / sin [tokens, rot / 2] or None; weight [dim] or None.
    Returns (y, the sum of the magnitudes that each value of y is the sum of)."""
    y = np.asarray(x, dtype=np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(weight, dtype=np.float64)
    mag = np.abs(y)
    if cos is None:
        return y, mag
    h = cos.shape[1]
    c, s = (np.asarray(t, dtype=np.float64)[:, None, :] for t in (cos, sin))
    out, big = y.copy(), mag.copy()
    lo, hi = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    a, b = y[..., lo], y[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    big[..., lo], big[..., hi] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return out, big


def code_groups(x, fmt):
    """64-bit x [..., dim] -> (codes, scale bytes).  The nearest code is searched among all of them, a tie
    goes to the even one."""
    g = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    nan = np.isnan(g).any(-1)
    g = np.where(nan[..., None], 0.0, g)
    amax = np.abs(g).max(-1)
    _, E = np.frexp(np.where(np.isinf(amax), 2.0**128, amax))
    top, mags = (8, oracle.e4m3_values()[:127].astype(np.float64)) if fmt == "mxfp8" else (2, E2M1)
    e = np.where(amax > 0, np.clip(E - 1 - top, -127, 127), -127)
    m = np.minimum(np.abs(g) * np.exp2(-e.astype(np.float64))[..., None], mags[-1])
    hi = np.searchsorted(mags, m)
    lo = np.maximum(hi - 1, 0)
    up, down = mags[hi] - m, m - mags[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    scales = np.where(nan, 255, e + 127).astype(np.uint8)
    if fmt == "mxfp8":
        return (code | (np.signbit(g).astype(np.uint8) << 7)).reshape(x.shape), scales
    nib = (code | ((g < 0).astype(np.uint8) << 3)).reshape(x.shape)
    return nib[..., 0::2] | (nib[..., 1::2] << 4), scales


def values(codes, scales, fmt):
    """What cache rows stand for, in 64 bits."""
    if fmt == "mxfp8":
        v = oracle.e4m3_values().astype(np.float64)[codes]
    else:
        v = E2M1_BOTH[np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])]
    two = np.exp2(scales.astype(np.float64) - 127)
    two = np.where(scales == 255, np.nan, two)
    return (v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32) * two[..., None]).reshape(v.shape)


def attention(q, k, v, scale):
    """One sequence: q [heads, dim], k and v [n, kv_heads, dim].  Returns (out, lse, sum_j p_j |v_j|,
    the largest sum over d of scale |q_d k_jd|), in 64 bits."""
    heads, dim = q.shape
    n, kvh, _ = k.shape
    if n == 0:
        z = np.zeros((heads, dim))
        return z, np.full(heads, -np.inf), z, np.zeros(heads)
    g = heads // kvh
    q = np.asarray(q, dtype=np.float64).reshape(kvh, g, dim)
    s = np.einsum("hgd,nhd->hgn", q, k) * scale
    size = np.einsum("hgd,nhd->hgn", np.abs(q), np.abs(k)).max(-1) * abs(scale)
    top = s.max(-1, keepdims=True)
    p = np.exp(s - top)
    total = p.sum(-1, keepdims=True)
    p = p / total
    out = np.einsum("hgn,nhd->hgd", p, v)
    mag = np.einsum("hgn,nhd->hgd", p, np.abs(v))
    lse = (top + np.log(total))[..., 0]
    return out.reshape(heads, dim), lse.reshape(heads), mag.reshape(heads, dim), size.reshape(heads)
