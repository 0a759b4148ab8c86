"""Rotary positions and sampling in 64 bits (numpy), from their definitions."""
import numpy as np

U = 2.0 ** -24


def features(pairs, order):
    """(a, b) features of each pair"""
    P, out, at = sum(pairs), [], 0
    for n in pairs:
        for j in range(n):
            i = len(out)
            out.append([(i, P + i), (2 * i, 2 * i + 1), (at + j, at + n + j)][order])
        at += 2 * n
    return out


def rope(x, pos, pairs, freqs, order):
    """x [B,S,H,D], pos [axes,B,S] -> rotated in 64 bits"""
    x = x.astype(np.float64)
    y = x.copy()
    axis = [a for a, n in enumerate(pairs) for _ in range(n)]
    for i, (a, b) in enumerate(features(pairs, order)):
        t = np.asarray(pos[axis[i]]).astype(np.longdouble) * np.longdouble(freqs[i])
        c, s = (f(t).astype(np.float64)[:, :, None] for f in (np.cos, np.sin))
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def rope_bound(x, pairs, order, out16):
    """how far each value may be off, by pairs: sine and cosine by 3 2^-24 (the angle's 2^-31 turns, its conversion, the
    product with 2 pi 2^-32 and that constant, half a step each of at most pi / 4, the polynomials' 2^-28 and the last fma's
    half step: 2.7), of |a| + |b|; the product b s and the fma half a step each of what they give. An fp16 output: half a
    step, or half of its smallest number."""
    x = np.abs(x.astype(np.float64))
    tol, mag = np.zeros_like(x), x.copy()
    for a, b in features(pairs, order):
        mag[..., a] = mag[..., b] = x[..., a] + x[..., b]
        tol[..., a] = tol[..., b] = 5 * U * mag[..., a]
    return tol + (2.0 ** -11 * mag + 2.0 ** -25 if out16 else 0)


def weights(x, temp):
    """weights of a row of logits relative to the largest's; None: no draw"""
    x = x.astype(np.float64)
    if np.isnan(x).any():
        return None
    m = x.max()
    if m == -np.inf:
        return None
    w = np.zeros(len(x))
    if not temp > 0:
        w[int(np.argmax(x))] = 1
        return w
    same = x == m
    live = np.isfinite(x) & ~same & (m < np.inf)        # beside an infinity nothing else weighs
    with np.errstate(all="ignore"):
        w[live] = np.exp((x[live] - m) / np.float64(temp))
    w[same] = 1
    return w


def kept(x, temp=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """weights of the kept tokens of a row, 0 elsewhere"""
    w = weights(x, temp)
    if w is None or not temp > 0:
        return w
    V = len(w)
    order = np.argsort(-(x.astype(np.float64) + 0.0), kind="stable")
    n = V if top_k <= 0 or top_k >= V else top_k
    run = np.cumsum(w[order])
    if top_p < 1:
        n = min(n, max(1, 1 + int((run[:n - 1] < np.float64(top_p) * run[n - 1]).sum())))
    if min_p > 0:
        n = min(n, int((w[order] >= min(np.float64(min_p), 1.0)).sum()))
    out = np.zeros(V)
    out[order[:n]] = w[order[:n]]
    return out


def sample(x, u, **kw):
    """(id, probability) of a row; with the distance of u from the nearest border between two tokens"""
    w = kept(x, **kw)
    if w is None:
        return -1, np.nan if np.isnan(x.astype(np.float64)).any() else 0.0, 1.0
    run = np.cumsum(w)
    at = min(max(float(u), 0.0), 1.0) * run[-1]
    i = int(np.searchsorted(run, at, side="right"))
    i = min(i, int(np.nonzero(w)[0][-1]))
    near = np.abs(run - at).min() / run[-1]
    return i, w[i] / run[-1], near
