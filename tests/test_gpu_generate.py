"""GPU parity of the operators of token-by-token generation: attention under masks, the 8-bit key / value
cache, attention over it, and what is done to logits, each against its definition in 64 bits
(tests/gen_oracle.py, which derives the tolerances)."""
import numpy as np
import pytest

import edge_maskgit_amd as ema
from tests import gen_oracle as ref

pytestmark = pytest.mark.gpu
F16, F32, F64, I32 = np.float16, np.float32, np.float64, np.int32


@pytest.fixture(scope="module")
def ctx():
    c = ema.Context(0)
    yield c
    c.close()


class Dev:
    """device buffers of one test, freed at its end"""

    def __init__(self, ctx):
        self.ctx, self.bufs = ctx, []

    def up(self, x, dtype=None):
        if x is None:
            return None
        b = self.ctx.upload(np.asarray(x) if dtype is None else np.asarray(x).astype(dtype))
        self.bufs.append(b)
        return b

    def get(self, b, shape, dtype):
        return self.ctx.download(b, shape, dtype)

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.ctx.sync()
        for b in self.bufs:
            self.ctx.free(b)


def close(got, want, tol, rel):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"NaN in {np.isnan(got).sum()} places, not in {np.isnan(want).sum()}"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    got, want = got[ok], want[ok]
    err = np.abs(got - want) - rel * np.abs(want)
    assert not err.size or err.max() <= tol, f"off by {err.max():.3g}, bound {tol:.3g}"


def qkv(rng, B, Sq, Sk, H, Hkv, D, spread=1.5):
    q = (rng.standard_normal((B, Sq, H, D)) * spread).astype(F16)
    k = rng.standard_normal((B, Sk, Hkv, D)).astype(F16)
    v = (rng.standard_normal((B, Sk, Hkv, D)) + 0.3).astype(F16)
    return q, k, v


def docs_of(rng, B, S, n, pad=0):
    out = np.full((B, S), -1, I32)
    for b in range(B):
        cuts = np.sort(rng.integers(0, S - pad + 1, n - 1))
        for d, (lo, hi) in enumerate(zip(np.r_[0, cuts], np.r_[cuts, S - pad])):
            out[b, lo:hi] = d
    return out


def run_masked(ctx, q, k, v, in16=True, out16=True, fill=7.0, **kw):
    """contiguous [B,S,H,D] inputs through mgh_attn_masked"""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1:3]
    t = F16 if in16 else F32
    with Dev(ctx) as dev:
        o = dev.up(np.full(q.shape, fill, F16 if out16 else F32))
        args = {n: dev.up(kw.get(n), d) for n, d in (("slopes", F32), ("prefix", I32), ("docs", I32))}
        ctx.attn_masked(dev.up(q, t), dev.up(k, t), dev.up(v, t), (1, H * D, D, Sq * H * D), (1, Hkv * D, D, Sk * Hkv * D), D, Sq,
                        Sk, H, Hkv, B, kw.get("scale", D ** -0.5), in16=in16, cap=kw.get("cap", 0.0), causal=kw.get("causal", False),
                        doc_stride=Sk, o_strides=(1, H * D, D, Sq * H * D), **{"o16" if out16 else "o": o}, **args)
        return dev.get(o, q.shape, F16 if out16 else F32)


def check_masked(ctx, q, k, v, in16=True, out16=True, **kw):
    scale = kw.setdefault("scale", q.shape[3] ** -0.5)
    got = run_masked(ctx, q, k, v, in16, out16, **kw)
    args = {n: kw[n] for n in ("cap", "slopes", "causal", "prefix", "docs") if n in kw}
    want = ref.masked(q, k, v, scale, **args)
    tol, rel = ref.bound(q, k, v, scale, kw.get("cap", 0.0), kw.get("slopes"), out16)
    close(got, want, tol, rel)
    return got


# B, Sq, Sk, H, Hkv, D: lengths from one token on, odd ones, fewer and more queries than keys
SHAPES = [(1, 1, 1, 1, 1, 16), (2, 1, 33, 4, 2, 32), (1, 5, 5, 3, 3, 48), (2, 17, 64, 4, 1, 64), (1, 63, 65, 2, 2, 80),
          (1, 130, 130, 3, 1, 96), (1, 40, 300, 6, 2, 112), (2, 65, 257, 4, 4, 128), (1, 257, 257, 2, 1, 48), (1, 9, 4, 2, 1, 64),
          (1, 3, 700, 12, 2, 128), (3, 2, 1, 2, 1, 16)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["full", "causal", "prefix", "docs", "causal-docs", "cap", "slopes", "all"])
def test_masked_attention(ctx, shape, kind):
    print(f"masked {shape} {kind}", flush=True)
    B, Sq, Sk, H, Hkv, D = shape
    rng = np.random.default_rng(sum(shape) + len(kind))
    q, k, v = qkv(rng, B, Sq, Sk, H, Hkv, D)
    kw = {}
    if kind in ("causal", "prefix", "causal-docs", "all"):
        kw["causal"] = True
    if kind in ("prefix", "all"):
        kw["prefix"] = np.array([(b + 1) * Sk // 3 for b in range(B)], I32)
    if kind in ("docs", "causal-docs", "all"):
        kw["docs"] = docs_of(rng, B, Sk, 3, pad=Sk // 8)
    if kind in ("cap", "all"):
        kw["cap"] = 2.5
    if kind in ("slopes", "all"):
        kw["slopes"] = (2.0 ** -np.arange(1, H + 1)).astype(F32)
    check_masked(ctx, q, k, v, **kw)
    check_masked(ctx, q, k, v, out16=False, **kw)


@pytest.mark.parametrize("shape", [(1, 70, 70, 2, 1, 48), (2, 1, 130, 4, 4, 64)])
def test_masked_attention_fp32_rows(ctx, shape):
    B, Sq, Sk, H, Hkv, D = shape
    rng = np.random.default_rng(5)
    q, k, v = (x.astype(F32) + rng.standard_normal(x.shape).astype(F32) * 1e-3 for x in qkv(rng, *shape))
    for out16 in (False, True):
        check_masked(ctx, q, k, v, in16=False, out16=out16, causal=True, slopes=np.full(H, 0.1, F32))


def test_masked_attention_sees_nothing(ctx):
    """padding queries, queries before the first key, no keys at all: rows of zeros"""
    rng = np.random.default_rng(3)
    q, k, v = qkv(rng, 1, 70, 70, 2, 2, 32)
    docs = np.full((1, 70), -1, I32)
    docs[0, 10:20] = 4
    got = check_masked(ctx, q, k, v, docs=docs)
    assert np.array_equal(got[0, :10], np.zeros_like(got[0, :10])) and np.array_equal(got[0, 20:], np.zeros_like(got[0, 20:]))
    got = check_masked(ctx, q, k[:, :30], v[:, :30], causal=True)
    assert not got[0, :40].any() and got[0, 40:].any()
    for out16 in (True, False):
        assert not run_masked(ctx, q, k[:, :0], v[:, :0], out16=out16).any()


@pytest.mark.parametrize("out16", [True, False])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("S", [33, 200, 700])
def test_masked_places_may_hold_anything(ctx, bad, out16, S):
    """keys and values that a row does not see do not reach it; rows that see one are as the formula"""
    rng = np.random.default_rng(S)
    q, k, v = qkv(rng, 1, S, S, 4, 2, 48)
    docs = docs_of(rng, 1, S, 3, pad=5)
    last = S - 3                                     # padding
    k[0, last], v[0, last] = bad, bad
    check_masked(ctx, q, k, v, out16=out16, docs=docs)
    at = S // 2                                      # seen by the rows from it on
    v[0, at, 1, 7] = bad
    check_masked(ctx, q, k, v, out16=out16, causal=True, docs=np.zeros_like(docs), **({"slopes": np.full(4, 0.01, F32)} if S == 33 else {}))
    k[0, at, 0, 3] = bad
    got = run_masked(ctx, q, k, v, out16=out16, causal=True)
    assert np.isfinite(got[0, :at].astype(F64)).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("D", [48, 128])
def test_padded_batch_of_anything(ctx, bad, D):
    """documents and padding behind them whose keys and values are never written; rows that see an infinity or
    NaN come out NaN, the rest as if it were not there"""
    rng = np.random.default_rng(16)
    q, k, v = qkv(rng, 2, 260, 260, 4, 2, D)
    docs = docs_of(rng, 2, 260, 3, pad=77)
    k[:, 183:] = bad
    v[:, 183:] = bad
    for kw in ({}, {"causal": True}, {"cap": 5.0}, {"slopes": np.full(4, 0.1, F32)}):
        for out16 in (False, True):
            got = check_masked(ctx, q, k, v, out16=out16, docs=docs, **kw)
            assert np.isfinite(got.astype(F64)).all() and not got[:, 183:].any()
    got = run_masked(ctx, q, k, v, causal=True)
    assert np.isfinite(got[:, :183].astype(F64)).all() and np.isnan(got[:, 183:].astype(F64)).all()


def test_masked_attention_scores_of_any_size(ctx):
    """a row whose scores climb, fall, or stand far above or below zero; a negative scale; scale 0"""
    rng = np.random.default_rng(8)
    q, k, v = qkv(rng, 1, 40, 500, 2, 2, 64)
    ramp = np.linspace(-6, 6, 500, dtype=F16)[None, :, None, None]
    for kk in (k + ramp, k - ramp, k * F16(8)):
        kk = kk.astype(F16)
        for scale in (1.0, -1.0, 0.0, 0.125):
            for out16 in (False, True):
                check_masked(ctx, np.abs(q), kk, v, scale=scale, out16=out16)
                check_masked(ctx, np.abs(q), kk, v, scale=scale, cap=30.0, out16=out16)


@pytest.mark.parametrize("scale", [-1e30, 1e30, -1e36])
def test_scores_far_from_zero(ctx, scale):
    """every score of a row below -1e31 (or above): a row that sees keys is no row that sees nothing. Dot products
    are 32 or 64, so weights are 0 or equal whatever the rounding; all keys of a block have one scale of codes."""
    rng = np.random.default_rng(15)
    q = np.ones((1, 3, 2, 32), F16)
    k = np.ones((1, 96, 1, 32), F16)
    k[0, ::3] = 2
    v = (rng.standard_normal((1, 96, 1, 32)) + 0.3).astype(F16)
    some = np.arange(96) % 3 == 0 if scale > 0 else np.arange(96) % 3 != 0
    for sk in (96, 70):
        for out16 in (False, True):
            for kw in ({}, {"causal": True}, {"slopes": np.zeros(2, F32)}):
                got = run_masked(ctx, q, k[:, :sk], v[:, :sk], out16=out16, scale=scale, **kw)
                for i in range(3):
                    n = sk - 2 + i if kw.get("causal") else sk
                    want = v[0, :n, 0].astype(F64)[some[:n]].mean(0)
                    close(got[0, i], np.stack([want] * 2), *ref.bound(q, k, v, 0.0, out16=out16))
    with Dev(ctx) as dev:
        c = Cache(dev, 1, 1, 32, 3, rng)
        c.append(k, v, [0])
        for out16 in (False, True):
            got = c.attend(q, [93], [3], out16=out16, scale=scale)
            for i in range(3):
                want = ref.cache_values(v[0])[:94 + i, 0][some[:94 + i]].mean(0)
                close(got[0, i], np.stack([want] * 2), *ref.bound(q, k, v, 0.0, out16=out16))


@pytest.mark.parametrize("cap", [60.0, 70.0, 1e4, 1e8])
def test_caps_of_any_size(ctx, cap):
    """scores far below the cap keep their relative accuracy"""
    rng = np.random.default_rng(14)
    q, k, v = qkv(rng, 1, 20, 150, 2, 1, 32)
    for slopes in (None, np.full(2, 0.05, F32)):
        check_masked(ctx, q, k, v, cap=cap, out16=False, causal=True, slopes=slopes)
        check_masked(ctx, q, k, v, cap=cap, scale=-0.3, slopes=slopes)
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, [150], [2], 2, 1, 32)
        check_cache(c, q, k, v, [150], [2], have, cap=cap, out16=False)


@pytest.mark.parametrize("D,G", [(48, 1), (64, 4), (128, 1), (128, 2)])
@pytest.mark.parametrize("kind", ["full", "docs", "causal", "cap", "slopes"])
def test_masked_attention_many_rows(ctx, D, G, kind):
    """enough rows for every plan (two row tiles per wave, several workgroups per CU): some rows against 64 bits"""
    print(f"many rows {D} {G} {kind}", flush=True)
    rng = np.random.default_rng(D + G)
    B, S, Hkv = 4, 1100, 8
    q, k, v = qkv(rng, B, S, S, Hkv * G, Hkv, D)
    docs = docs_of(rng, B, S, 4, pad=70)
    kw = {"docs": {"docs": docs}, "causal": {"causal": True, "prefix": np.array([0, 5, 700, 1100], I32)}, "cap": {"cap": 9.0},
          "slopes": {"slopes": (0.5 ** np.arange(Hkv * G)).astype(F32)}}.get(kind, {})
    for out16 in (True, False):
        got = run_masked(ctx, q, k, v, out16=out16, **kw)
        assert np.isfinite(got).all()
        tol, rel = ref.bound(q, k, v, D ** -0.5, kw.get("cap", 0.0), kw.get("slopes"), out16)
        for i in (0, 63, 64, 127, 128, 500, 1029, 1030, 1099):
            b, h = int(rng.integers(B)), int(rng.integers(Hkv * G))
            j = np.arange(S)
            seen = np.ones(S, bool)
            if kind == "causal":
                seen = (j <= i) | (j < kw["prefix"][b])
            if kind == "docs":
                seen = (docs[b] == docs[b, i]) & (docs[b] >= 0)
            sl = kw.get("slopes")
            want = ref.attention_row(q[b, i, h].astype(F64), k[b, :, h // G].astype(F64), v[b, :, h // G].astype(F64), D ** -0.5,
                                     kw.get("cap", 0.0), None if sl is None else float(sl[h]), i, seen)
            close(got[b, i, h], want, tol, rel)


def test_masked_attention_a_million_keys(ctx):
    """more keys than a workgroup notes documents of, and rows in parts of a long sequence"""
    rng = np.random.default_rng(15)
    Sq, Sk, D = 26000, 1100000, 16
    q, k, v = (rng.standard_normal((1, n, 1, D)).astype(F16) for n in (Sq, Sk, Sk))
    docs = np.sort(rng.integers(0, 30, (1, Sk)).astype(I32), 1)
    docs[0, -50:] = -1
    got = run_masked(ctx, q, k, v, docs=docs, causal=True)
    few = run_masked(ctx, q[:, -60:], k, v, docs=docs, causal=True)
    tol, rel = ref.bound(q, k, v, D ** -0.5, out16=True)
    j = np.arange(Sk)
    for i in (0, 1, 12345, Sq - 60, Sq - 51, Sq - 50, Sq - 1):
        p = Sk - Sq + i
        seen = (j <= p) & (docs[0] == docs[0, p]) & (docs[0] >= 0)
        want = ref.attention_row(q[0, i, 0].astype(F64), k[0, :, 0].astype(F64), v[0, :, 0].astype(F64), D ** -0.5, 0.0, None, p, seen)
        close(got[0, i, 0], want, tol, rel)
        if i >= Sq - 60:
            close(few[0, i - (Sq - 60), 0], want, tol, rel)


def _put(ctx, ptr, x):
    x = np.ascontiguousarray(x)
    ctx._check(ema.lib().mgh_h2d(ctx.h, ptr, x.ctypes.data, x.nbytes))


def test_offsets_past_32_bits(ctx):
    """rows, sequences and pages whose byte offsets do not fit 32 bits"""
    rng = np.random.default_rng(16)
    B, S, H, D = 2, 300, 2, 64
    q, k, v = qkv(rng, B, S, S, H, H, D)
    want = run_masked(ctx, q, k, v, causal=True)
    token, seq = 1 << 22, (1 << 22) * 300 + 64                # 8 MiB between rows, 2.5 GB per sequence
    with Dev(ctx) as dev:
        big = ctx.alloc(2 * (seq * B + (1 << 20)))
        dev.bufs.append(big)
        for b in range(B):
            for i in range(S):
                _put(ctx, big.ptr + 2 * (b * seq + i * token), np.concatenate([q[b, i].ravel(), k[b, i].ravel(), v[b, i].ravel()]))
        st = (1, token, D, seq)
        o = dev.up(np.zeros_like(q))
        ctx.attn_masked(big, big.ptr + 2 * H * D, big.ptr + 4 * H * D, st, st, D, S, S, H, H, B, D ** -0.5, causal=True, o16=o,
                        o_strides=(1, H * D, D, S * H * D))
        assert np.array_equal(dev.get(o, q.shape, F16), want)
    with Dev(ctx) as dev:
        lens, new, Hkv = [70, 40], [2, 1], 8
        c, q, k, v, have = cache_case(dev, rng, lens, new, 8, Hkv, 128)
        want = c.attend(q, lens, new)
        pages = 80000                                          # 2.6 GB of codes each
        per = Hkv * 32 * 128
        dk, dv, ds = ctx.alloc(pages * per), ctx.alloc(pages * per), ctx.alloc(pages * Hkv * 8)
        dev.bufs += [dk, dv, ds]
        c.k, c.v, c.scales, c.pages = dk, dv, ds, pages
        c.set_table((79990 + np.arange(2 * c.nb).reshape(2, c.nb) * 3 % 10).astype(I32))
        c.append(k[:, :max(have)], v[:, :max(have)], [0, 0], have)
        assert np.array_equal(c.attend(q, lens, new), want)
        rk, _ = c.read(have, 72)
        assert np.array_equal(rk[0, :, :64], ref.cache_values(k[0, :64]).astype(F32).transpose(1, 0, 2))


def test_masked_attention_strides(ctx):
    """any strides and alignments give what contiguous rows give: views of a fused row, heads outside
    the tokens, features apart, odd offsets, one row for all sequences, separate output layouts"""
    rng = np.random.default_rng(4)
    B, S, H, Hkv, D = 2, 77, 4, 2, 32
    q, k, v = qkv(rng, B, S, S, H, Hkv, D)
    want = run_masked(ctx, q, k, v, causal=True)
    want32 = run_masked(ctx, q, k, v, causal=True, out16=False)
    w = (H + 2 * Hkv) * D
    for pad in (0, 8, 3):
        rows = np.zeros((B, S, w + pad), F16)
        rows[:, :, :w] = np.concatenate([x.reshape(B, S, -1) for x in (q, k, v)], 2)
        with Dev(ctx) as dev:
            r, o = dev.up(rows), dev.up(np.zeros((B, H, S, D), F32))
            st = (1, w + pad, D, S * (w + pad))
            ctx.attn_masked(r.ptr, r.ptr + 2 * H * D, r.ptr + 2 * (H + Hkv) * D, st, st, D, S, S, H, Hkv, B, D ** -0.5, o=o,
                            causal=True)                        # contiguous {D, S, H, B} output
            assert np.array_equal(dev.get(o, (B, H, S, D), F32).transpose(0, 2, 1, 3), want32), pad
    with Dev(ctx) as dev:                                       # features outermost, 2-byte offset
        flat = [dev.up(np.r_[F16(0), np.ascontiguousarray(x.transpose(3, 0, 2, 1)).ravel()]) for x in (q, k, v)]
        o = dev.up(np.zeros((B, S, H, D + 1), F16))
        ctx.attn_masked(flat[0].ptr + 2, flat[1].ptr + 2, flat[2].ptr + 2, (B * H * S, 1, S, H * S), (B * Hkv * S, 1, S, Hkv * S), D, S,
                        S, H, Hkv, B, D ** -0.5, o16=o, causal=True, o_strides=(1, H * (D + 1), D + 1, S * H * (D + 1)))
        got = dev.get(o, (B, S, H, D + 1), F16)
        assert np.array_equal(got[..., :D], want) and not got[..., D].any()
    with Dev(ctx) as dev:                                       # the same keys for both sequences
        one = run_masked(ctx, q, np.stack([k[0], k[0]]), np.stack([v[0], v[0]]), causal=True)
        dq, dk, dv, o = dev.up(q), dev.up(k[0]), dev.up(v[0]), dev.up(np.zeros_like(q))
        st = (1, H * D, D, S * H * D)
        ctx.attn_masked(dq, dk, dv, st, (1, Hkv * D, D, 0), D, S, S, H, Hkv, B, D ** -0.5, o16=o, causal=True, o_strides=st)
        assert np.array_equal(dev.get(o, q.shape, F16), one)


# ---- the cache ----------------------------------------------------------------------------


class Cache:
    """a cache on the device with pages in any order, everything not yet written set to what must not matter"""

    def __init__(self, dev, B, Hkv, D, max_blocks, rng, spare=2):
        self.dev, self.B, self.Hkv, self.D, self.nb = dev, B, Hkv, D, max_blocks
        self.pages = B * max_blocks + spare
        self.table = rng.permutation(self.pages)[:B * max_blocks].reshape(B, max_blocks).astype(I32)
        n = self.pages * Hkv * 32 * D
        assert n == ema.kv8_code_bytes(self.pages, Hkv, D) and self.pages * Hkv * 8 == ema.kv8_scale_bytes(self.pages, Hkv)
        assert B * Hkv * 64 * D * 2 == ema.kv8_tail_bytes(B, Hkv, D)
        self.k, self.v = dev.up(np.full(n, 255, np.uint8)), dev.up(np.full(n, 255, np.uint8))
        self.scales = dev.up(np.full(self.pages * Hkv * 2, np.nan, F32))
        tail = np.full(B * Hkv * 64 * D, np.nan, F16)
        self.kt, self.vt = dev.up(tail), dev.up(tail)
        self.set_table(self.table)

    def set_table(self, table):
        self.dtable = self.dev.up(table)
        self.h = ema.Kv8(self.k, self.v, self.scales, self.kt, self.vt, self.dtable, self.nb, self.pages, self.Hkv, self.D, self.B)

    def append(self, k, v, lens, new=None, in16=True):
        """k, v [B,S,Hkv,D]"""
        S, w = k.shape[1], self.Hkv * self.D
        t = F16 if in16 else F32
        self.dev.ctx.kv8_append(self.h, self.dev.up(k, t), self.dev.up(v, t), (1, w, self.D, S * w), S, self.dev.up(lens, I32),
                                self.dev.up(new, I32), in16=in16)

    def state(self):
        g = self.dev.get
        n = self.pages * self.Hkv * 32 * self.D
        return (g(self.k, n, np.uint8), g(self.v, n, np.uint8), g(self.scales, self.pages * self.Hkv * 2, F32),
                g(self.kt, self.B * self.Hkv * 64 * self.D, F16), g(self.vt, self.B * self.Hkv * 64 * self.D, F16))

    def read(self, lens, n, first=None, f16=False):
        t = F16 if f16 else F32
        shape = (self.B, self.Hkv, n, self.D)
        k, v = self.dev.up(np.full(shape, 9, t)), self.dev.up(np.full(shape, 9, t))
        self.dev.ctx.kv8_read(self.h, self.dev.up(first, I32), n, self.dev.up(lens, I32), **({"k16": k, "v16": v} if f16 else {"k": k, "v": v}))
        return self.dev.get(k, shape, t), self.dev.get(v, shape, t)

    def attend(self, q, lens, new=None, in16=True, out16=True, fill=7.0, cap=0.0, slopes=None, scale=None):
        """q [B,S,H,D]"""
        _, S, H, D = q.shape
        st = (1, H * D, D, S * H * D)
        o = self.dev.up(np.full(q.shape, fill, F16 if out16 else F32))
        self.dev.ctx.kv8_attn(self.h, self.dev.up(q, F16 if in16 else F32), st, S, self.dev.up(lens, I32), self.dev.up(new, I32), H,
                              D ** -0.5 if scale is None else scale, in16=in16, cap=cap, slopes=self.dev.up(slopes, F32), o_strides=st,
                              **{"o16" if out16 else "o": o})
        return self.dev.get(o, q.shape, F16 if out16 else F32)


def tokens(rng, B, n, Hkv, D):
    k = (rng.standard_normal((B, n, Hkv, D)) * np.exp(0.7 * rng.standard_normal((1, 1, Hkv, D)))).astype(F16)
    v = rng.standard_normal((B, n, Hkv, D)).astype(F16)
    k[:, 5:6], v[:, 40:50, :, :D // 2] = 0, 0
    return k, v


@pytest.mark.parametrize("D,Hkv", [(16, 1), (48, 3), (64, 2), (80, 1), (128, 2)])
def test_cache_holds_the_definition(ctx, D, Hkv):
    """whole blocks exactly as the rule's codes and scales, byte for byte; the rest as it came"""
    rng = np.random.default_rng(D)
    B, n = 2, 101
    k, v = tokens(rng, B, n, Hkv, D)
    lens = [n, 64]
    with Dev(ctx) as dev:
        c = Cache(dev, B, Hkv, D, 4, rng)
        c.append(k, v, [0, 0], lens)
        gk, gv, gs, _, _ = c.state()
        gs = gs.reshape(c.pages, Hkv, 2)
        for b in range(B):
            for i in range(lens[b] // 32):
                for h in range(Hkv):
                    pg = c.table[b, i]
                    at = slice((pg * Hkv + h) * 32 * D, (pg * Hkv + h + 1) * 32 * D)
                    ck, dk = ref.quantize(k[b, 32 * i:32 * i + 32, h])
                    cv, dv = ref.quantize(v[b, 32 * i:32 * i + 32, h])
                    assert gs[pg, h].tolist() == [dk, dv]
                    assert np.array_equal(gk[at], (ck + 128).astype(np.uint8).ravel())
                    assert np.array_equal(gv[at], ref.v_layout(cv))
        for f16 in (False, True):
            rk, rv = c.read(lens, n + 3, f16=f16)
            for got, x in ((rk, k), (rv, v)):
                for b in range(B):
                    want = ref.cache_values(x[b, :lens[b]]).astype(F32).astype(got.dtype)
                    assert np.array_equal(got[b, :, :lens[b]], want.transpose(1, 0, 2))
                    assert (got[b, :, lens[b]:] == 9).all()                 # rows past the end: as they were
        a, _ = c.read(lens, 40, first=[50, 60])
        b32, _ = c.read(lens, n)
        assert np.array_equal(a[0], b32[0, :, 50:90]) and np.array_equal(a[1, :, :4], b32[1, :, 60:64]) and (a[1, :, 4:] == 9).all()


def test_cache_does_not_depend_on_the_grouping(ctx):
    """token by token, in odd pieces, fp32 rows, ragged pieces of a padded batch: the same bytes; and a
    sequence shortened by up to 32 tokens goes on from there"""
    rng = np.random.default_rng(9)
    B, n, Hkv, D = 2, 150, 2, 48
    k, v = tokens(rng, B, n, Hkv, D)
    with Dev(ctx) as dev:
        def filled(steps, in16=True):
            c = Cache(dev, B, Hkv, D, 5, np.random.default_rng(1))
            done = np.zeros(B, int)
            for new in steps:
                new = np.minimum(new, n - done)
                S = max(int(new.max()), 1)
                kk, vv = np.full((2, B, S, Hkv, D), np.nan, F16)            # rows past a sequence's tokens are not read
                for b in range(B):
                    kk[b, :new[b]], vv[b, :new[b]] = k[b, done[b]:done[b] + new[b]], v[b, done[b]:done[b] + new[b]]
                c.append(kk, vv, done, new, in16)
                done = done + new
            assert (done == n).all()
            return c
        want = filled([np.array([n, n])]).state()
        for steps in ([np.array([1, 1])] * n, [np.array([7, 7])] * 30, [np.array([33, 40])] * 6, [np.array([0, 64]), np.array([90, 1])] * 10):
            for in16 in (True, False):
                got = filled(steps, in16).state()
                # the ring holds the last 64 tokens either way, the pool what was whole
                for x, y in zip(got, want):
                    assert np.array_equal(x, y, equal_nan=x.dtype != np.uint8)
        c = filled([np.array([n, n])])
        c.append(-k[:, 118:140], -v[:, 118:140], [118, 118])                # back by 32, other tokens
        k2, v2 = k.copy(), v.copy()
        k2[:, 118:140], v2[:, 118:140] = -k[:, 118:140], -v[:, 118:140]
        for got, x in zip(c.read([140, 140], 140), (k2, v2)):
            for b in range(B):
                assert np.array_equal(got[b], ref.cache_values(x[b, :140]).astype(F32).transpose(1, 0, 2))


def test_cache_advance(ctx):
    with Dev(ctx) as dev:
        lens = dev.up([5, 0, 70], I32)
        ctx.kv8_advance(lens, dev.up([1, 0, 3], I32), 3, 4)
        ctx.kv8_advance(lens, None, 3, 2)
        assert dev.get(lens, 3, I32).tolist() == [8, 2, 75]


def test_cache_of_values_next_to_the_border(ctx):
    """codes are the exact quotient's rounding: blocks whose values lie at and next to (n + 1/2) d, tiny
    ones, and ones whose scale is not the quotient in fp32"""
    rng = np.random.default_rng(2)
    D, Hkv, n = 16, 2, 64
    k = np.zeros((1, n, Hkv, D), F16)
    for blk, top in ((0, 127.0), (1, 100.0)):
        for h in range(Hkv):
            x = np.arange(512) * 0.5 - 128 if h == 0 else rng.integers(-254, 255, 512) * 0.5 * (top / 127)
            x = np.clip(x, -top, top).astype(F16)
            x[0] = F16(top)
            k[0, 32 * blk:32 * blk + 32, h] = x.reshape(32, D)
    v = (k * F16(2.0 ** -24)).astype(F16)                       # fp16's smallest numbers
    with Dev(ctx) as dev:
        c = Cache(dev, 1, Hkv, D, 2, rng)
        c.append(k, v, [0])
        for got, x in zip(c.read([n], n), (k, v)):
            assert np.array_equal(got[0], ref.cache_values(x[0]).astype(F32).transpose(1, 0, 2))


def cache_case(dev, rng, lens, new, H, Hkv, D, spare=1):
    B, S = len(lens), max(max(new), 1)
    have = [a + b for a, b in zip(lens, new)]
    nb = -(-max(have) // 32) + spare
    k, v = tokens(rng, B, max(max(have), 50), Hkv, D)
    c = Cache(dev, B, Hkv, D, nb, rng)
    c.append(k[:, :max(have)], v[:, :max(have)], [0] * B, have) if max(have) else None
    q = (rng.standard_normal((B, S, H, D)) * 1.5).astype(F16)
    return c, q, k, v, have


def check_cache(c, q, k, v, lens, new, have, out16=True, **kw):
    B, S, H, D = q.shape
    got = c.attend(q, lens, new, out16=out16, **kw)
    scale = kw.get("scale") or D ** -0.5
    for b in range(B):
        kk, vv = ref.cache_values(k[b, :have[b]])[None], ref.cache_values(v[b, :have[b]])[None]
        qq = q[b:b + 1, :new[b]].astype(F64)
        want = np.zeros((new[b], H, D))
        for i in range(new[b]):
            for h in range(H):
                g = h // (H // c.Hkv)
                sl = kw.get("slopes")
                want[i, h] = ref.attention_row(qq[0, i, h], kk[0, :, g], vv[0, :, g], scale, kw.get("cap", 0.0),
                                               None if sl is None else float(sl[h]), lens[b] + i, np.arange(have[b]) <= lens[b] + i)
        tol, rel = ref.bound(qq, kk, vv, scale, kw.get("cap", 0.0), kw.get("slopes"), out16)
        close(got[b, :new[b]], want, tol, rel)
        assert (got[b, new[b]:] == 7).all()                                 # rows past a sequence's tokens: as they were
    return got


CACHES = [([0], [1], 1, 1, 16), ([30, 31, 32], [1, 1, 1], 4, 4, 32), ([0, 63, 64, 95], [1, 1, 1, 1], 6, 2, 48),
          ([200, 3], [1, 1], 8, 1, 64), ([1000, 0, 517], [1, 1, 1], 4, 2, 128), ([40, 7], [5, 2], 4, 2, 80),
          ([100], [33], 3, 3, 96), ([10, 90, 0], [9, 0, 17], 8, 2, 112), ([2500], [1], 16, 2, 128), ([62, 66], [20, 20], 12, 1, 64)]


@pytest.mark.parametrize("lens,new,H,Hkv,D", CACHES)
@pytest.mark.parametrize("kind", ["plain", "cap", "slopes"])
def test_cache_attention(ctx, lens, new, H, Hkv, D, kind):
    print(f"cache {lens} {new} {H} {Hkv} {D} {kind}", flush=True)
    rng = np.random.default_rng(sum(lens) + D)
    kw = {"cap": {"cap": 3.0}, "slopes": {"slopes": (0.5 ** np.arange(1, H + 1)).astype(F32)}}.get(kind, {})
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, lens, new, H, Hkv, D)
        check_cache(c, q, k, v, lens, new, have, **kw)
        check_cache(c, q, k, v, lens, new, have, out16=False, **kw)


def test_cache_attention_fp32_queries_and_layouts(ctx):
    rng = np.random.default_rng(6)
    lens, new, H, Hkv, D = [70, 33], [3, 3], 4, 2, 32
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, lens, new, H, Hkv, D)
        want = c.attend(q, lens, new)
        assert np.array_equal(c.attend(q.astype(F32), lens, new, in16=False), want)
        # heads outside the tokens, features apart, an odd offset; a contiguous {D, S, H, B} output
        x = dev.up(np.r_[F16(0), np.ascontiguousarray(q.transpose(3, 0, 2, 1)).ravel()])
        o = dev.up(np.zeros((2, H, 3, D), F16))
        ctx.kv8_attn(c.h, x.ptr + 2, (2 * H * 3, 1, 3, H * 3), 3, dev.up(lens, I32), None, H, D ** -0.5, o16=o)
        assert np.array_equal(dev.get(o, (2, H, 3, D), F16).transpose(0, 2, 1, 3), want)


def test_cache_attention_tiny_and_large_values(ctx):
    """blocks whose scales lie far apart: each block's weights meet its own scale in fp32"""
    rng = np.random.default_rng(7)
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, [160], [1], 4, 2, 64)
        size = (2.0 ** np.array([-14, 9, -20, 0, 5, 3])).repeat(32)[:v.shape[1]]
        v = (v * size[None, :, None, None]).astype(F16)
        c.append(k[:, :161], v[:, :161], [0])
        check_cache(c, q, k, v, [160], [1], have, out16=False)


def test_cache_holds_infinities_as_nan(ctx):
    """a block with an infinity or NaN reads as NaN and reaches the rows that see it; tokens behind the last
    whole block keep what they are, and rows that do not see them yet are not reached"""
    rng = np.random.default_rng(10)
    lens, new = [96], [3]
    for bad in (np.nan, np.inf):
        with Dev(ctx) as dev:
            c, q, k, v, have = cache_case(dev, rng, lens, new, 2, 2, 32)
            k2, v2 = k.copy(), v.copy()
            v2[0, 98, 0, 3] = bad                                            # the last of three new tokens
            c.append(k2[:, :99], v2[:, :99], [0])
            got = c.attend(q, lens, new)
            clean = Cache(dev, 1, 2, 32, 4, np.random.default_rng(0))
            clean.append(k[:, :99], v[:, :99], [0])
            want = clean.attend(q, lens, new)
            # rows may be taken by another path there, whose weights are not rounded to fp16: each within its
            # bound of the 64-bit value, so within twice the bound of one another
            tol, rel = (2 * x for x in ref.bound(q, k, v, 32 ** -0.5, out16=True))
            close(got[0, :2], want[0, :2], tol, rel)
            close(got[0, 2, 1], want[0, 2, 1], tol, rel)
            assert not np.isfinite(got[0, 2, 0, 3]) and np.isfinite(got[0, 2, 0, 4])
            v2 = v.copy()
            v2[0, 40, 1, 3] = bad
            c.append(k[:, :99], v2[:, :99], [0])
            rk, rv = c.read([99], 99)
            assert np.isnan(rv[0, 1, 32:64]).all() and np.isfinite(rv[0, 0]).all() and np.isfinite(rk).all()
            got = c.attend(q, lens, new)
            close(got[0, :, 0], want[0, :, 0], tol, rel)
            assert np.isnan(got[0, :, 1]).all()


def test_cache_refuses_bad_numbers_on_the_device(ctx):
    """page numbers outside the pool, negative lengths, too many tokens, past the table: nothing is written,
    rows read as NaN, other sequences are not touched by it"""
    rng = np.random.default_rng(11)
    lens, new, H, Hkv, D = [70, 70, 70, 70], [1, 1, 1, 1], 2, 1, 32
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, lens, new, H, Hkv, D)
        want, before = c.attend(q, lens, new), c.state()
        good = c.table
        table = good.copy()
        table[0, 1], table[1, 0] = c.pages, -1                              # whole blocks that the rows need
        table[2, 2:] = -7                                                   # the open block and those after it: not read
        c.set_table(table)
        got = c.attend(q, lens, new)
        assert np.isnan(got[:2]).all() and np.array_equal(got[2:], want[2:])
        rk, rv = c.read([71] * 4, 71)
        assert np.isnan(rk[0, :, 32:64]).all() and np.isfinite(rk[0, :, :32]).all() and np.isnan(rv[1, :, :32]).all()
        assert np.isfinite(rk[2:]).all()
        c.set_table(good)
        bad = [-1, 32 * c.nb, 70, 70]
        n = [1, 1, 2, -1]                                                   # S is 1
        got = c.attend(q, bad, n)
        assert np.isnan(got).all()
        c.append(k[:, :1], v[:, :1], bad, n)
        for x, y in zip(c.state(), before):
            assert np.array_equal(x, y, equal_nan=x.dtype != np.uint8)
        assert np.isnan(c.read([-1, 32 * c.nb + 1, 71, 71], 5)[0][:2]).all()
        assert np.array_equal(c.attend(q, lens, new), want)


def test_cache_table_wider_than_the_sequences(ctx):
    """parts that most sequences have no blocks for, short and long ones in a batch, more rows than a workgroup's"""
    rng = np.random.default_rng(17)
    with Dev(ctx) as dev:
        lens, new = [5, 300, 0, 1700], [1, 1, 1, 1]
        c, q, k, v, have = cache_case(dev, rng, lens, new, 8, 2, 64, spare=900)
        check_cache(c, q, k, v, lens, new, have)
        c, q, k, v, have = cache_case(dev, rng, [400, 90], [40, 30], 8, 2, 128, spare=200)
        check_cache(c, q, k, v, [400, 90], [40, 30], have, cap=5.0)
        check_cache(c, q, k, v, [400, 90], [40, 30], have, out16=False, slopes=np.full(8, 0.2, F32))


@pytest.mark.parametrize("B,nb", [(64, 8), (64, 300)])
def test_cache_attention_large_batches(ctx, B, nb):
    """a workgroup per CU and more, sequences past and below the length that is taken in parts"""
    rng = np.random.default_rng(nb)
    Hkv, D, H = 4, 48, 4
    with Dev(ctx) as dev:
        lens = rng.integers(0, 32 * nb - 1, B)
        lens[:2] = 32 * nb - 1, 0
        pages = B * nb
        k, v = rng.standard_normal((2, 1, 32 * nb, Hkv, D)).astype(F16)
        c = Cache(dev, 1, Hkv, D, nb, rng, spare=0)
        c.append(k, v, [0])
        # every sequence reads the same pages; its open block is its own
        table = np.repeat(c.table, B, 0)
        one = c
        c = Cache(dev, B, Hkv, D, nb, rng, spare=0)
        c.k, c.v, c.scales, c.pages = one.k, one.v, one.scales, one.pages
        tk, tv = np.full((B, Hkv, 64, D), np.nan, F16), np.full((B, Hkv, D, 64), np.nan, F16)
        for b, n in enumerate(lens):
            t = np.arange((n + 1) // 32 * 32, n + 1)
            tk[b][:, t % 64], tv[b][:, :, t % 64] = k[0, t].transpose(1, 0, 2), v[0, t].transpose(1, 2, 0)
        c.kt, c.vt = dev.up(tk), dev.up(tv)
        c.set_table(table)
        q = rng.standard_normal((B, 1, H, D)).astype(F16)
        got = c.attend(q, lens)
        whole = ref.cache_values(k[0]), ref.cache_values(v[0])
        tol, rel = ref.bound(q, whole[0][None], whole[1][None], D ** -0.5, out16=True)
        for b in list(range(6)) + [B - 1]:
            n = int(lens[b]) + 1
            cut = n // 32 * 32
            kk = np.concatenate([whole[0][:cut], k[0, cut:n].astype(F64)])
            vv = np.concatenate([whole[1][:cut], v[0, cut:n].astype(F64)])
            for h in range(H):
                want = ref.attention_row(q[b, 0, h].astype(F64), kk[:, h], vv[:, h], D ** -0.5, 0.0, None, n - 1, np.ones(n, bool))
                close(got[b, 0, h], want, tol, rel)


def test_cache_pages_shared(ctx):
    """two sequences that share a whole block of the same tokens"""
    rng = np.random.default_rng(12)
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, [60, 60], [1, 1], 2, 1, 64)
        k[1, :32], v[1, :32] = k[0, :32], v[0, :32]
        c.append(k[:, :61], v[:, :61], [0, 0])
        table = c.table.copy()
        table[1, 0] = table[0, 0]
        want = c.attend(q, [60, 60])
        c.set_table(table)
        assert np.array_equal(c.attend(q, [60, 60]), want)


# ---- logits -------------------------------------------------------------------------------


def check_logits(ctx, x, place=False, **kw):
    """at most four roundings to fp32 of values no larger than `mag`, and one to x's type"""
    rows, V = x.shape
    want, mag = ref.logits(x, **kw)
    with Dev(ctx) as dev:
        dx = dev.up(x)
        y = dx if place else dev.up(np.full(x.shape, 3, x.dtype))
        kinds = (("hist", I32), ("hist_len", I32), ("rep", F32), ("freq", F32), ("pres", F32), ("bias", F32), ("allowed", np.uint32))
        args = {n: dev.up(kw.get(n), t) for n, t in kinds}
        b, m = kw.get("bias"), kw.get("allowed")
        ctx.logits_process(dx, rows, V, y, f16=x.dtype == F16, max_hist=0 if kw.get("hist") is None else kw["hist"].shape[1],
                           bias_stride=V if b is not None and len(b) > 1 else 0,
                           allowed_stride=m.shape[1] if m is not None and len(m) > 1 else 0, **args)
        got = dev.get(y, x.shape, x.dtype).astype(F64)
    with np.errstate(all="ignore"):
        there = want.astype(x.dtype)                     # (past the type's largest number: infinite)
    odd = ~np.isfinite(there)
    assert np.array_equal(got[odd], there[odd].astype(F64), equal_nan=True)
    ok = ~odd
    half = 2.0 ** -11 * np.abs(want[ok]) + 2.0 ** -25 if x.dtype == F16 else 0
    assert (np.abs(got[ok] - want[ok]) <= 5 * 2.0 ** -24 * mag[ok] + half).all()


@pytest.mark.parametrize("rows,V", [(1, 1), (1, 33), (3, 2025), (2, 4096), (2, 4097), (5, 20001), (1, 131072)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_logits(ctx, rows, V, dtype):
    rng = np.random.default_rng(rows + V)
    x = (rng.standard_normal((rows, V)) * 4).astype(dtype)
    hist = rng.integers(0, max(V // 3, 1), (rows, 500)).astype(I32)
    hist[:, ::50] = rng.choice([-1, V, 2 ** 31 - 1, -2 ** 31], hist[:, ::50].shape)      # ids outside count nowhere
    lens = rng.integers(0, 501, rows).astype(I32)
    pen = dict(hist=hist, hist_len=lens, rep=(1 + rng.random(rows)).astype(F32), freq=rng.random(rows).astype(F32),
               pres=rng.random(rows).astype(F32))
    bias = rng.standard_normal((rows, V)).astype(F32)
    allowed = rng.integers(0, 2 ** 32, (rows, (V + 31) // 32)).astype(np.uint32)
    for place in (False, True):
        check_logits(ctx, x, place, **pen, bias=bias, allowed=allowed)
    check_logits(ctx, x, **pen)
    check_logits(ctx, x, bias=bias[:1])
    check_logits(ctx, x, allowed=allowed[:1])
    check_logits(ctx, x, hist=hist, rep=pen["rep"])
    check_logits(ctx, x, hist=hist, pres=pen["pres"], hist_len=np.array([-3] + [900] * (rows - 1), I32))
    check_logits(ctx, x)


def test_logits_special_values(ctx):
    """infinities, NaN, the lowest numbers, and rows whose mask leaves nothing"""
    low = np.finfo(F32).min
    x = np.array([[0.0, -0.0, np.inf, -np.inf, np.nan, low, -low, 1.0]], F32).repeat(3, 0)
    hist = np.arange(8, dtype=I32)[None].repeat(3, 0)
    bias = np.array([[0, 0, 0, 0, 0, 0, low, low]], F32)
    allowed = np.array([[0xff], [0], [0x0f]], np.uint32)
    with np.errstate(all="ignore"):
        check_logits(ctx, x, hist=hist, rep=np.array([2, 1.5, 1], F32), allowed=allowed)
        check_logits(ctx, x, bias=bias, allowed=allowed)


def test_logits_strides(ctx):
    """rows apart: what lies between them stays as it was; a history for all rows"""
    rng = np.random.default_rng(1)
    rows, V, w = 3, 1001, 1040
    for dtype in (F32, F16):
        x = rng.standard_normal((rows, w)).astype(dtype)
        hist = rng.integers(0, V, 40).astype(I32)
        with Dev(ctx) as dev:
            dx, dy = dev.up(x), dev.up(np.full((rows, w + 3), 5, dtype))
            ctx.logits_process(dx, rows, V, dy, f16=dtype == F16, x_stride=w, y_stride=w + 3, hist=dev.up(hist), hist_stride=0,
                               max_hist=40, pres=dev.up(np.full(rows, 2, F32)))
            got = dev.get(dy, (rows, w + 3), dtype)
            want, _ = ref.logits(x[:, :V], hist=hist[None].repeat(rows, 0), pres=np.full(rows, 2, F32))
            assert np.array_equal(got[:, :V], want.astype(F32).astype(dtype)) and (got[:, V:] == 5).all()


# ---- together -----------------------------------------------------------------------------


def test_generating_token_by_token(ctx):
    """prompt -> masked attention and cache, then one token after another over the cache, with the head's
    logits edited and the best token taken; the steps captured once and replayed. Against the same steps in
    64 bits (with the cache's values as its definition gives them)."""
    rng = np.random.default_rng(21)
    B, P, T, V, H, Hkv, D = 2, 37, 30, 96, 4, 2, 16
    E = H * D
    w = (H + 2 * Hkv) * D
    table_q = (rng.standard_normal((V, w)) * 0.8).astype(F32)          # a token's q, k, v
    head = (rng.standard_normal((V, E))).astype(F32)
    prompt = rng.integers(0, V, (B, P)).astype(I32)
    plen = np.array([P, 20], I32)
    docs = np.where(np.arange(P)[None] < plen[:, None], 0, -1).astype(I32)
    allowed = np.full((B, 3), 0xfffffff0, np.uint32)
    rows16 = table_q.astype(F16)
    st, ost = (1, w, D, w * P), (1, E, D, E * P)
    with Dev(ctx) as dev:
        c = Cache(dev, B, Hkv, D, 3, rng)
        x = dev.up(rows16[prompt])
        o = dev.up(np.zeros((B, P, E), F16))
        ctx.attn_masked(x.ptr, x.ptr + 2 * E, x.ptr + 2 * (E + Hkv * D), st, st, D, P, P, H, Hkv, B, D ** -0.5, causal=True,
                        docs=dev.up(docs), doc_stride=P, o16=o, o_strides=ost)
        got_prompt = dev.get(o, (B, P, H, D), F16)
        lens = dev.up(np.zeros(B, I32))
        ctx.kv8_append(c.h, x.ptr + 2 * E, x.ptr + 2 * (E + Hkv * D), st, P, lens, dev.up(plen))
        ctx.kv8_advance(lens, dev.up(plen), B, P)
        # a step on the device: rows of the newest tokens, cache, attention, head, logits
        rows, att = dev.up(np.zeros((B, w), F32)), dev.up(np.zeros((B, E), F32))
        lg, y = dev.up(np.zeros((B, V), F32)), dev.up(np.zeros((B, V), F32))
        dt, dh, ids = dev.up(table_q), dev.up(head), dev.up(np.zeros(B, I32))
        hist, hlen = dev.up(np.zeros((B, T), I32)), dev.up(np.zeros(B, I32))
        pres, allow = dev.up(np.full(B, 0.7, F32)), dev.up(allowed)
        st1, ost1 = (1, w, D, w), (1, E, D, E)

        def step():
            ctx.get_rows(dt, w, V, ids, B, rows)
            ctx.kv8_append(c.h, rows.ptr + 4 * E, rows.ptr + 4 * (E + Hkv * D), st1, 1, lens, in16=False)
            ctx.kv8_attn(c.h, rows, st1, 1, lens, None, H, D ** -0.5, in16=False, o=att, o_strides=ost1, cap=20.0)
            ctx.gemm_f32(dh, V, E, att, B, None, 0, None, lg)
            ctx.logits_process(lg, B, V, y, hist=hist, max_hist=T, hist_len=hlen, pres=pres, allowed=allow, allowed_stride=3)
            ctx.kv8_advance(lens, None, B, 1)

        tok = np.array([prompt[b, plen[b] - 1] for b in range(B)], I32)
        seqs = [list(prompt[b, :plen[b]]) for b in range(B)]
        past = [[] for _ in range(B)]
        graph = None
        for t in range(T):
            ctx.write(ids, tok)
            ctx.write(hist, np.array([p + [0] * (T - len(p)) for p in past], I32))
            ctx.write(hlen, np.array([len(p) for p in past], I32))
            if t == 1:
                ctx.graph_begin()
                step()
                graph = ctx.graph_end()
            graph.launch() if graph else step()
            got, got_lens = dev.get(y, (B, V), F32), dev.get(lens, B, I32)
            assert got_lens.tolist() == [plen[b] + t + 1 for b in range(B)]
            for b in range(B):
                seqs[b].append(int(tok[b]))
                f = rows16[seqs[b]].astype(F64)
                n = len(seqs[b])
                kk = ref.cache_values(f[:, E:E + Hkv * D].reshape(n, Hkv, D).astype(F16))
                vv = ref.cache_values(f[:, E + Hkv * D:].reshape(n, Hkv, D).astype(F16))
                q = f[-1, :E].reshape(H, D)
                a = np.stack([ref.attention_row(q[h], kk[:, h // 2], vv[:, h // 2], D ** -0.5, 20.0, None, n - 1, np.ones(n, bool))
                              for h in range(H)])
                tol, rel = ref.bound(q[None, None], kk[None], vv[None], D ** -0.5, 20.0)
                want = head.astype(F64) @ a.ravel()
                room = np.abs(head).sum(1).max() * (tol + 2.0 ** -20 * np.abs(a).max()) + 1e-6
                one, _ = ref.logits(want[None], hist=np.array([past[b] + [0]], I32), hist_len=[len(past[b])], pres=[0.7], allowed=allowed[b:b + 1])
                assert np.array_equal(np.isneginf(got[b]), np.isneginf(one[0]))
                live = np.isfinite(one[0])
                assert np.abs(got[b][live] - one[0][live]).max() <= room
                past[b].append(int(tok[b]))
                tok[b] = int(np.argmax(got[b]))
        graph.destroy()
    tol, rel = ref.bound(*(rows16[prompt][:, :, a:a + n * D].reshape(B, P, n, D) for a, n in ((0, H), (E, Hkv), (E + Hkv * D, Hkv))), D ** -0.5, out16=True)
    full = rows16[prompt]
    want = ref.masked(full[:, :, :E].reshape(B, P, H, D), full[:, :, E:E + Hkv * D].reshape(B, P, Hkv, D),
                      full[:, :, E + Hkv * D:].reshape(B, P, Hkv, D), D ** -0.5, causal=True, docs=docs)
    close(got_prompt, want, tol, rel)


def test_capture_and_replay(ctx):
    """each operator captured, replayed with eager work between, two contexts' streams side by side"""
    rng = np.random.default_rng(31)
    q, k, v = qkv(rng, 1, 3, 900, 8, 2, 64)
    with Dev(ctx) as dev, ema.Context(0) as other:
        st, kst = (1, 512, 64, 3 * 512), (1, 128, 64, 900 * 128)
        o, o2 = dev.up(np.zeros((1, 3, 8, 64), F16)), dev.up(np.zeros((1, 3, 8, 64), F16))
        dq, dk, dv = dev.up(q), dev.up(k), dev.up(v)
        c, cq, ck, cv, have = cache_case(dev, rng, [700], [2], 8, 2, 64)
        lens, dcq = dev.up([700], I32), dev.up(cq)
        co = dev.up(np.zeros(cq.shape, F32))
        cst = (1, 512, 64, 1024)

        def work(cx, out):
            cx.attn_masked(dq, dk, dv, st, kst, 64, 3, 900, 8, 2, 1, 0.125, causal=True, o16=out, o_strides=st)

        def cache():
            ctx.kv8_attn(c.h, dcq, cst, 2, lens, None, 8, 0.125, o=co, o_strides=cst)

        work(ctx, o)
        cache()
        want, cwant = dev.get(o, q.shape, F16), dev.get(co, cq.shape, F32)
        ctx.graph_begin()
        work(ctx, o)
        cache()
        g = ctx.graph_end()
        work(other, o2)
        other.sync()
        for rep in range(4):
            ctx.write(o, np.zeros(q.shape, F16))
            ctx.write(co, np.zeros(cq.shape, F32))
            g.launch()
            work(other, o2)
            if rep % 2:
                cache()                                    # eager between replays, the same workspace
            assert np.array_equal(dev.get(o, q.shape, F16), want) and np.array_equal(dev.get(co, cq.shape, F32), cwant)
            other.sync()
            assert np.array_equal(dev.get(o2, q.shape, F16), want)
        g.destroy()


def test_replay_after_the_workspaces_grew(ctx):
    """a graph captured in a context of its own keeps the buffers that it was captured with when later calls need
    larger ones, and two graphs of one context may take turns"""
    rng = np.random.default_rng(32)
    q, k, v = qkv(rng, 1, 2, 600, 4, 2, 64)
    Q, K, V = qkv(rng, 2, 40, 3000, 8, 4, 64)
    with ema.Context(0) as own, Dev(own) as dev:
        def call(x, in16):
            _, Sq, H, D = x[0].shape
            Sk, Hkv = x[1].shape[1:3]
            ins = [dev.up(a, F16 if in16 else F32) for a in x]
            o = dev.up(np.zeros(x[0].shape, F16))
            st, kst = (1, H * D, D, Sq * H * D), (1, Hkv * D, D, Sk * Hkv * D)

            def run():
                own.attn_masked(*ins, st, kst, D, Sq, Sk, H, Hkv, len(x[0]), D ** -0.5, o16=o, in16=in16, o_strides=st)
            return run, o, x[0].shape

        def capture(run):
            run()
            own.graph_begin()
            run()
            return own.graph_end()

        small, o1, s1 = call((q, k, v), False)                  # packed, in parts
        g1 = capture(small)
        want1 = dev.get(o1, s1, F16)
        large, o2, s2 = call((Q, K, V), False)
        g2 = capture(large)                                     # both buffers grow
        want2 = dev.get(o2, s2, F16)
        close(want1, ref.masked(q, k, v, 0.125), *ref.bound(q, k, v, 0.125, out16=True))
        for rep in range(3):
            for g, o, s, want in ((g1, o1, s1, want1), (g2, o2, s2, want2)):
                own.write(o, np.zeros(s, F16))
                g.launch()
                if rep == 1:
                    (small if g is g2 else large)()
                assert np.array_equal(dev.get(o, s, F16), want)
        g1.destroy()
        g2.destroy()
