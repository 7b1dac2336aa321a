"""The operators around drafted rows in float64 numpy, from their definitions,
row by row."""
import math

import numpy as np


def frequencies(rot_dim, theta, scaling=None):
    """(angle per position of each pair, factor on cosine and sine)."""
    s = scaling or {"kind": "plain"}
    i = np.arange(rot_dim // 2)
    f = float(theta) ** (-2.0 * i / rot_dim)
    if s["kind"] == "plain":
        return f, 1.0
    if s["kind"] == "linear":
        return f / s["factor"], 1.0
    turns = s["original"] * f / (2 * math.pi)
    if s["kind"] == "yarn":
        def pair(t):
            return rot_dim * math.log(s["original"] / (t * 2 * math.pi)) / (2 * math.log(theta))
        lo = max(0, math.floor(pair(s.get("beta_fast", 32.0))))
        hi = min(rot_dim - 1, math.ceil(pair(s.get("beta_slow", 1.0))))
        own = 1 - np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        mag = 0.1 * math.log(s["factor"]) + 1 if s["factor"] > 1 else 1.0
    else:
        low, high = s.get("low", 1.0), s.get("high", 4.0)
        own = np.clip((turns - low) / (high - low), 0, 1)
        mag = 1.0
    return f * own + f / s["factor"] * (1 - own), mag


def turned(x, pos, rot_dim, interleaved, freq, mag):
    """x [heads][hd] float64 at one position."""
    y = x.copy()
    a = slice(0, rot_dim, 2) if interleaved else slice(0, rot_dim // 2)
    b = slice(1, rot_dim, 2) if interleaved else slice(rot_dim // 2, rot_dim)
    c, s = np.cos(pos * freq) * mag, np.sin(pos * freq) * mag
    y[:, a] = x[:, a] * c - x[:, b] * s
    y[:, b] = x[:, b] * c + x[:, a] * s
    return y


def normed(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def path(parents, t):
    """The drafted rows that row t sees, itself included (None: a chain)."""
    if parents is None:
        return list(range(t + 1))
    rows = []
    while t >= 0:
        rows.append(t)
        t = int(parents[t])
    return rows


def stored(x, fmt):
    """What a format (0 f32, 1 f16, 2 int8) holds of f32 rows, as float32."""
    x = np.asarray(x, np.float32)
    if fmt == 0:
        return x
    if fmt == 1:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    wide = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        scale = (np.abs(wide).max(-1, keepdims=True) / 127).astype(np.float32)
        q = np.clip(np.rint(wide / scale.astype(np.float64)), -127, 127).astype(np.float32)
    q = np.where(scale == 0, np.float32(0), q)
    return np.where(np.isfinite(x).all(-1, keepdims=True), q * scale, np.float32(np.nan))


def attention(q, k, v, lens, counts, parents, scale):
    """q [n][rows][h][hd], k and v [n][positions][kvh][hd] as float64, the rows
    of sequence b at lens[b] ..; returns (out, bound): bound on what sums of
    products in f32 are off by, elementwise. The scores: products of the split
    query (parts of 11 bits: 2^-22) summed over hd terms; the probabilities: the
    exponent of a score off by d is off by e^d - 1, and so is their sum; the
    values: one more sum over the positions, and a few roundings."""
    n, rows, h, hd = q.shape
    g = h // k.shape[2]
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    u = 2.0 ** -24
    for b in range(n):
        for t in range(counts[b]):
            at = list(range(lens[b])) + [lens[b] + r for r in
                                         path(None if parents is None else parents[b], t)]
            for a in range(k.shape[2]):
                kk, vv = k[b, at, a], v[b, at, a]
                x = q[b, t, a * g:(a + 1) * g]
                s = x @ kk.T * scale
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[b, t, a * g:(a + 1) * g] = p @ vv
                size = np.abs(x) @ np.abs(kk).T * abs(scale)
                d = size.max(-1, keepdims=True) * (hd + 16) * u + np.abs(s).max(-1, keepdims=True) * 8 * u
                bound[b, t, a * g:(a + 1) * g] = \
                    (2 * d + (len(at) / 8 + 64) * u) * (p @ np.abs(vv)) * (1 + 2 * d)
    return out, bound


def scores(logits, tokens, top_k):
    """logits [rows][vocab] float32, tokens [rows][m]: (logprobs, entropy,
    top_ids, top_logprobs), a row with NaN, +inf or nothing finite: NaN."""
    z = logits.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = z.max(-1, keepdims=True)
        lse = m + np.log(np.exp(z - m).sum(-1, keepdims=True))
        lp = z - lse
        p = np.exp(lp)
        entropy = -np.where(p > 0, p * lp, 0).sum(-1)
    bad = ~np.isfinite(lse[:, 0])
    lp[bad] = np.nan
    entropy[bad] = np.nan
    ok = (tokens >= 0) & (tokens < z.shape[1])
    at = np.where(ok, tokens, 0)
    logprobs = np.where(ok, np.take_along_axis(lp, at, 1), np.nan)
    key = np.where(np.isnan(z), np.inf, -z)  # NaN last, of equal ones the lowest
    key = np.where(np.isnan(z), np.inf, key)
    order = np.lexsort((np.broadcast_to(np.arange(z.shape[1]), z.shape), key, np.isnan(z)), axis=-1)
    top = order[:, :top_k]
    return logprobs, entropy, top.astype(np.int32), np.take_along_axis(lp, top, 1)
