"""The operators of token-by-token generation in 64 bits (numpy), from their definitions."""
import numpy as np

BLOCK, RING = 32, 64


def attention_row(q, k, v, scale, cap, slope, p, seen):
    """one query row over keys [n, D]; `seen` [n] truth values"""
    if not seen.any():
        return np.zeros(v.shape[1])
    at = np.nonzero(seen)[0]
    s = (k[at] @ q) * scale
    if cap:
        s = cap * np.tanh(s / cap)
    if slope is not None:
        s = s - slope * np.abs(p - at)
    m = s.max()
    if m == -np.inf:
        return np.zeros(v.shape[1])
    w = np.exp(s - m)
    live = w > 0
    return (w[live] @ v[at[live]]) / w.sum()


def masked(q, k, v, scale, cap=0.0, slopes=None, causal=False, prefix=None, docs=None):
    """q [B,Sq,H,D], k and v [B,Sk,Hkv,D] -> [B,Sq,H,D]"""
    q, k, v = (x.astype(np.float16).astype(np.float64) for x in (q, k, v))
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1:3]
    out = np.zeros(q.shape)
    j = np.arange(Sk)
    for b in range(B):
        for i in range(Sq):
            p = Sk - Sq + i
            seen = np.ones(Sk, bool)
            if causal:
                seen = (j <= p) | (j < (prefix[b] if prefix is not None else 0))
            if docs is not None:
                seen = seen & (docs[b] == docs[b][p]) & (docs[b] >= 0) if p >= 0 else np.zeros(Sk, bool)
            for h in range(H):
                g = h // (H // Hkv)
                with np.errstate(all="ignore"):
                    out[b, i, h] = attention_row(q[b, i, h], k[b, :, g], v[b, :, g], scale, cap,
                                                 None if slopes is None else float(slopes[h]), p, seen)
    return out


def bound(q, k, v, scale, cap=0.0, slopes=None, out16=False):
    """how far an output may be from the 64-bit one, and the relative part of it.

    Scores: a dot product of D terms in fp32 is off by at most (D + 8) 2^-24 of the sum of its terms'
    magnitudes (the products of fp16 values are exact), the cap's tanh by 8 2^-24 cap (exp2, reciprocal
    and fma, 1-2 ulp each; from a cap of 64 on small arguments by their series, 8 2^-24 of the score), and each of the few operations on a score of magnitude S by 2^-24 S. That
    difference is the relative error of a weight, with 2^-20 for its exponential and the 22 bits of it
    that meet v. Sums of n weights and products add n 2^-24. An output is a ratio of such sums: twice
    that, of the largest |v|. With fp16 outputs the weights are rounded to fp16 (2^-11) and the output is
    once more."""
    q, k, v = (np.abs(x.astype(np.float16).astype(np.float64)) for x in (q, k, v))
    q, k, v = (np.where(np.isfinite(x), x, 0) for x in (q, k, v))
    D, n = q.shape[-1], k.shape[1]
    mag = abs(scale) * (q.reshape(-1, D).max(0) * k.reshape(-1, D).max(0)).sum() if k.size and q.size else 0.0
    far = 0.0 if slopes is None else float(np.abs(slopes).max()) * max(n, q.shape[1])
    top = (min(mag, cap) if cap else mag) + far
    eps = 2.0 ** -24 * ((D + 8) * mag + 8 * (cap if cap <= 64 else min(4 * cap, 4 * mag)) + 6 * top + n) + 2.0 ** -20
    vmax = v.max() if v.size else 0.0
    # (2^-30: outputs below fp16's normal numbers are rounded to multiples of 2^-24)
    return 2 * (eps + (2.0 ** -11 if out16 else 0)) * vmax + (2.0 ** -25 if out16 else 1e-30), 2.0 ** -11 if out16 else 2.0 ** -24


def row_tolerance(q, k, v, scale, cap=0.0, slope=None, p=0, seen=None, out16=False):
    """how far each feature of one row (q [D], keys [n, D], a finite row that sees something) may be from
    attention_row's, to first order, from the row's own terms.

    Score j: products of fp16 values are exact in fp32; the matrix unit may lose a whole step (2^-23) per
    addition of the sum of the terms that are not zero, of their magnitudes. Scaling it, with the constants'
    own roundings, is four roundings (2^-24). The cap is six of the cap (tanh = 1 - 2 r, r = 1 / (e + 1), at
    x = s / cap >= 1/4: r itself one, e's step and its argument's two roundings 2 r (1 - r) of theirs, at most 0.94
    and 0.9, the sum e + 1 0.75, the last fma and the constant one each, together 5.6, below that no more), or where
    |x| < 3/4 ten of the score; with an fp16 output up to a cap of 64 the former throughout. The slope and the
    subtraction of the reference (within 15 log2 units of the maximum) are one each of what they give. A weight's
    exponential is off by a step, and hi + lo in fp16 by 2^-22 of it (fp16: 2^-11), with 2^-32 of the row's largest
    weight where lo leaves fp16's normal numbers. An error e_j of the weights p_j (sum 1) moves the output by
    sum p_j e_j (v_j - o). The sums: a step per addition that a term goes through, of the terms' magnitudes (64 keys,
    hi and lo, at a time, then chunk by chunk, waves and parts)."""
    seen = np.ones(len(k), bool) if seen is None else seen
    at = np.nonzero(seen)[0]
    k, v, a = k[at], v[at], abs(float(scale))
    u = 2.0 ** -24
    terms = k * q
    raw, mag, nnz = a * np.abs(terms.sum(1)), a * np.abs(terms).sum(1), (terms != 0).sum(1)
    s = terms.sum(1) * scale
    e = 2 * u * np.maximum(nnz - 1, 0) * mag + 4 * u * raw
    if cap:
        small = (np.abs(s) < 0.74 * cap) & (not out16 or cap > 64)
        s = cap * np.tanh(s / cap)
        e = e + np.where(small, 10 * u * np.abs(s), 6 * u * cap)
    if slope is not None:
        far = np.abs(slope) * np.abs(p - at)
        s = s - slope * np.abs(p - at)
        e = e + 2 * u * far + u * np.abs(s)
    w = np.exp(s - s.max())
    w, live = w / w.sum(), w.sum()
    e = e + u * (np.abs(s) + np.abs(s - s.max()) + 15 * np.log(2)) + 2 * u + (2.0 ** -11 if out16 else 2.0 ** -22)
    o = w @ v
    depth = 2 * min(len(at), 64) + len(at) / 64 + min(len(at) / 8, 16) + 2
    tol = (w * e) @ np.abs(v - o) + (2.0 ** -32 * len(at) / live + 2 * u * depth) * (w @ np.abs(v) + np.abs(o))
    return 1.01 * tol + 4 * u * np.abs(o) + (2.0 ** -11 * np.abs(o) + 2.0 ** -25 if out16 else 1e-30)


def quantize(x):
    """codes [-127, 127] and the scale of one block (any shape) of fp16 values"""
    top = np.abs(x).max()
    d = np.float32(top) / np.float32(127)
    if not d > 0 or not np.isfinite(d):
        return np.zeros(x.shape, np.int64), d
    t = np.abs(x.astype(np.float64)) / np.float64(d)
    c = np.floor(t)
    c = c + (t - c >= 0.5)
    return (np.sign(x) * c).astype(np.int64), d


def cache_values(k):
    """what the cache holds of tokens [n, Hkv, D] (fp16 values): whole blocks quantized, the rest as it is"""
    out = k.astype(np.float16).astype(np.float64)
    for t in range(0, k.shape[0] // BLOCK * BLOCK, BLOCK):
        for h in range(k.shape[1]):
            c, d = quantize(k[t:t + BLOCK, h].astype(np.float16))
            out[t:t + BLOCK, h] = c * np.float64(d) if np.isfinite(d) else np.nan
    return out


def v_layout(codes):
    """codes [32, D] -> the bytes of a block of V"""
    t, d = np.meshgrid(np.arange(BLOCK), np.arange(codes.shape[1]), indexing="ij")
    out = np.zeros(codes.size, np.uint8)
    out[((d // 2) * 4 + t // 8) * 16 + (d % 2) * 8 + t % 8] = codes + 128
    return out


def logits(x, hist=None, hist_len=None, rep=None, freq=None, pres=None, bias=None, allowed=None):
    """x [rows, V] -> edited logits in 64 bits and the magnitude that its roundings go by"""
    y = x.astype(np.float64)
    rows, V = y.shape
    mag = np.abs(y)
    if hist is not None:
        for r in range(rows):
            n = hist.shape[1] if hist_len is None else min(max(int(hist_len[r]), 0), hist.shape[1])
            ids = hist[r, :n]
            count = np.bincount(ids[(ids >= 0) & (ids < V)], minlength=V).astype(np.float64)
            a = 1.0 if rep is None else float(rep[r])
            f = 0.0 if freq is None else float(freq[r])
            p = 0.0 if pres is None else float(pres[r])
            off = f * count + p
            z = np.where(y[r] > 0, y[r] / a, y[r] * a)
            mag[r] = np.where(count > 0, np.abs(z) + np.abs(off), mag[r])
            y[r] = np.where(count > 0, z - off, y[r])
    if bias is not None:
        y = y + bias.astype(np.float64)
        mag = mag + np.abs(bias)
    if allowed is not None:
        v = np.arange(V)
        y = np.where((allowed[:, v // 32] >> (v % 32)) & 1, y, -np.inf)
    return y, mag
