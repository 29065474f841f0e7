"""A plain 8-bit cache in NumPy, 64 bits where it computes: what the tests of QuantKVCache compare with."""

import numpy as np
import torch

TREE16 = [-1, 0, 0, 0, 0, 1, 1, 2, 2, 3, 3, 4, 4, 5, 5, 6]


def codes(x, scheme):
    """(codes as float32, scale) of heads x (.., d) in fp32: the definition."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        top = np.max(np.abs(x), -1, keepdims=True)
        good = np.all(np.isfinite(x), -1, keepdims=True)
        scale = (np.where(top > 0, top, np.float32(1)) / np.float32(127 if scheme == "int8" else 448)).astype(np.float32)
        scale = np.maximum(scale, np.float32(2.0 ** -126))
        y = np.where(good, x / scale, 0).astype(np.float32)
    if scheme == "int8":
        c = np.clip(np.rint(y), -127, 127)
    else:
        c = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).float().numpy()
    return c.astype(np.float32), np.where(good, scale, np.float32(np.nan))


def in_8_bits(x, scheme):
    c, s = codes(x, scheme)
    return (c * s).astype(np.float32)


def depth_and_seen(parents, n):
    """(depth [n], seen [n, n]); parents None: a chain."""
    if parents is None:
        return np.arange(n), np.tril(np.ones((n, n), bool))
    depth, seen = np.zeros(n, int), np.eye(n, dtype=bool)
    for i, p in enumerate(parents[:n]):
        if p >= 0:
            depth[i] = depth[p] + 1
            seen[i] |= seen[p]
    return depth, seen


def heads_in(x, w, eps, turn, cos, sin, interleaved):
    """Norm and rotation of heads x (rows, heads, d), positions turn (rows,), in 64 bits."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w
    if cos is None:
        return x
    n = cos.shape[1]
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    c, s = np.asarray(cos, np.float64)[turn][:, None], np.asarray(sin, np.float64)[turn][:, None]
    y = x.copy()
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    return y


def attention(q, k, v, n_com, depth, seen, window, scale):
    """(out, weight) of one entry: q (n, H, d); k, v (n_com + n, KH, d) as the cache holds them.  weight (n, H, d): sum of p |v|, and
    (n, H, 3): the largest sum of |q k| times scale, the largest |v| of the head, and the largest of sum |q| times max |k| times scale, over
    what a row sees."""
    n, H, d = q.shape
    KH = k.shape[1]
    out, weight, reach = np.zeros((n, H, d)), np.zeros((n, H, d)), np.zeros((n, H, 3))
    for i in range(n):
        see = np.concatenate([np.ones(n_com, bool), seen[i]])
        if window:
            at = np.concatenate([np.arange(n_com), n_com + depth])
            see &= (n_com + depth[i]) - at < window
        if not see.any():
            continue
        for h in range(H):
            g = h // (H // KH)
            kk, vv, qq = k[see, g].astype(np.float64), v[see, g].astype(np.float64), q[i, h].astype(np.float64)
            a = kk @ qq * scale
            e = np.exp(a - a.max())
            p = e / e.sum()
            out[i, h], weight[i, h] = p @ vv, p @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(qq)).max() * scale, np.abs(vv).max(), np.abs(qq).sum() * np.abs(kk).max() * scale
    return out, weight, reach


def tolerance(out, weight, reach, d, keys, dtype, int8=False):
    """What rounding may cost.  Scores: queries in two halves of 11 bits (2^-22 of a term), products of 16 channels summed in 32 bits, at
    most d / 16 partial sums and a few products behind them, each at most 2^-23 of the sum of the magnitudes `reach` (a unit off,
    not half: matrix instructions may cut).  A weight is off by twice that (its own score and the maximum) and 2^-21 for the exponential; the
    sums over keys by 2^-23 for every 16 keys and every merge of parts, at most keys / 16 + 64 in all.  bf16 results: weights in
    11 bits (2^-12 each way: 2^-11 in all) and half a step of the result, 2^-8 of it, taken from a value that is itself off.
    Small weights: p s (s: scale of a value) is held as a half of p s 2^15 / R with R < 2 max s, whose smallest step is 2^-24; half of
    it is 2^-40 R of a weight, and times a code of at most max|v| / max s that is 2^-39 max|v| for every key (the sum of p is 1 or more).
    bf16 rows in numbers of more than 16 have p s 2^11 / R there, with R < 8 max s: half the smallest step is 2^-36 R, so 2^-33 max|v| for
    every key, and p is relative to a maximum at most 2^4 too low, so that the sum of p is still 1 or more.
    bf16 rows with int8 codes (int8 true): sums may begin at -1152 sum q' and take in codes that are 1152 too large, so that what they
    pass through is at most (1152 + 1152 + 127) sum|q'| times the scale of the key, max|k| / 127: 2431 / 127 < 20 times sum|q| max|k|."""
    reach, top, wide = reach[..., 0], reach[..., 1], reach[..., 2]
    score = 2.0 ** -22 * reach + 2.0 ** -23 * (d / 16 + 8) * (20 * wide if int8 and dtype == "bf16" else reach)
    rel = 2 * score + 2.0 ** -21 + 2.0 ** -22 * (keys / 16 + 64) + (2.0 ** -11 if dtype == "bf16" else 0.0)
    t = rel[..., None] * weight * 2 + ((2.0 ** -33 if dtype == "bf16" else 2.0 ** -39) * keys * top)[..., None]      # numerator and denominator
    return t + (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24) * (np.abs(out) + t) + 1e-30
