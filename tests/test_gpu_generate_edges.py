"""Token-by-token generation where it can go wrong: infinities that a row sees, rows whose sums leave fp16,
keys whose weight is zero, sequences that a call refuses among good ones with few and many parts. Against the
definitions in 64 bits (tests/gen_oracle.py)."""
import numpy as np
import pytest

from tests import gen_oracle as ref
from tests.test_gpu_generate import Cache, Dev, cache_case, check_cache, check_masked, close, ctx, qkv, run_masked, tokens  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, F64, I32 = np.float16, np.float32, np.float64, np.int32


# ---- the cache's lengths ------------------------------------------------------------------


def test_cache_advance_leaves_refused_sequences_refused(ctx):
    """numbers that append and attention refuse do not become a length that they take"""
    rng = np.random.default_rng(1)
    bad, new, S = [70, 70, -1, -1, 2 ** 31 - 1, 5], [2, -1, 0, 1, 1, 1], 1
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, [70] * 6, [1] * 6, 2, 1, 32)
        before = c.state()
        lens = dev.up(bad, I32)
        ctx.kv8_advance(lens, dev.up(new, I32), 6, S)
        assert dev.get(lens, 6, I32).tolist() == [70, 70, -1, -1, 2 ** 31 - 1, 6]
        idle = dev.up([-1, -5, 70], I32)
        ctx.kv8_advance(idle, None, 3, 4)                                   # idle slots stay idle
        assert dev.get(idle, 3, I32).tolist() == [-1, -5, 74]
        # four refused steps in a row: no byte of the pages and rings changes, every row is NaN
        lens = dev.up([70, 70, -1, -1, 2 ** 31 - 1, 32 * c.nb], I32)
        fresh = dev.up([2, -1, 1, 1, 1, 1], I32)
        st, w = (1, 32, 32, 32), dev.up(rng.standard_normal((6, 1, 1, 32)), F16)
        o, qst, dq = dev.up(np.zeros((6, 1, 2, 32), F32)), (1, 64, 32, 64), dev.up(q)
        for _ in range(4):
            ctx.kv8_append(c.h, w, w, st, S, lens, fresh)
            ctx.kv8_attn(c.h, dq, qst, S, lens, fresh, 2, 0.2, o=o, o_strides=qst)
            assert np.isnan(dev.get(o, (6, 2, 32), F32)).all()
            ctx.kv8_advance(lens, fresh, 6, S)
        for x, y in zip(c.state(), before):
            assert np.array_equal(x, y, equal_nan=x.dtype != np.uint8)


# ---- infinities that a row sees -----------------------------------------------------------


@pytest.mark.parametrize("D", [16, 48, 64, 80, 112, 128])
@pytest.mark.parametrize("in16", [True, False])
def test_open_block_with_infinite_keys(ctx, D, in16):
    """a key behind the last whole block with an infinite feature (fp32 ones from 65520 on are): its score is an
    infinity, so it weighs nothing where that is the negative one, whatever the width of the heads"""
    rng = np.random.default_rng(D)
    lens, new, H, Hkv = [40, 3], [4, 2], 4, 2
    big = F32(np.inf) if in16 else F32(65520)
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, lens, new, H, Hkv, D)
        q[..., 0], q[..., 7] = np.abs(q[..., 0]) + F16(0.1), -np.abs(q[..., 7]) - F16(0.1)
        k = k.astype(F32)
        k[0, 36, 0, 0], k[0, 41, :, 7], k[1, 1, 1, 0], k[1, 3, 0, 7] = -big, big, -big, big
        c.append(k[:, :max(have)], v[:, :max(have)], [0, 0], have, in16)
        with np.errstate(over="ignore"):
            k = k.astype(F16)
        assert np.isinf(k).sum() == 5
        for out16 in (True, False):
            for kw in ({}, {"slopes": np.full(H, 0.1, F32)}, {"cap": 30.0}):
                got = check_cache(c, q, k, v, lens, new, have, out16=out16, **kw)
                assert all(np.isfinite(got[b, :new[b]].astype(F64)).all() for b in range(2))


@pytest.mark.parametrize("out16", [True, False])
def test_capped_scores_of_infinite_keys(ctx, out16):
    """the cap of an infinite product is -cap, also for a row that sees nothing else in a chunk of 64 keys"""
    rng = np.random.default_rng(3)
    q, k, v = qkv(rng, 1, 200, 200, 2, 1, 48)
    q[..., 3] = np.abs(q[..., 3]) + F16(0.1)
    docs = np.zeros((1, 200), I32)
    for first in (63, 127, 61):                       # a document begins with the last keys of a chunk
        docs[:, first:] += 1
        k[0, first:(first // 64 + 1) * 64, 0, 3] = -np.inf
    for cap in (5.0, 30.0):
        check_masked(ctx, q, k, v, out16=out16, cap=cap, docs=docs)
        check_masked(ctx, q, k, v, out16=out16, cap=cap, docs=docs, causal=True)


@pytest.mark.parametrize("out16", [True, False])
def test_scores_past_the_reach_of_the_reference(ctx, out16):
    """scores of 2e8, where fp32 numbers lie 16 apart: weights against a reference that could not be set closer leave
    fp16, and a later chunk far above takes the whole weight"""
    rng = np.random.default_rng(4)
    D = 16
    q, k = np.zeros((1, 2, 2, D), F16), np.zeros((1, 320, 1, D), F16)
    q[..., 0], q[..., 1] = 32768, 0.25
    v = (rng.standard_normal((1, 320, 1, D)) + 0.3).astype(F16)
    for i, n in ((0, 2), (1, 4), (2, 127)):
        k[0, 64 * i:64 * i + 64, 0, :2] = 127, n
    got = run_masked(ctx, q, k[:, :192], v[:, :192], out16=out16, scale=32.0)
    close(got[0], np.broadcast_to(v[0, 128:192, 0].astype(F64).mean(0), got[0].shape), *ref.bound(q, k, v, 0.0, out16=out16))
    k[:] = 0
    for i, n in ((0, 2), (4, 4), (8, 127)):           # blocks of one wave, in a batch of whole sequences; codes are the values
        k[0, 32 * i:32 * i + 32, 0, :2] = 127, n
    B = 256
    with Dev(ctx) as dev:
        c = Cache(dev, B, 1, D, 10, rng)
        c.append(k.repeat(B, 0), v.repeat(B, 0), [0] * B)
        want = ref.cache_values(v[0])[256:288, 0].mean(0)
        got = c.attend(q.repeat(B, 0), [318] * B, [2] * B, out16=out16, scale=32.0)
        close(got, np.broadcast_to(want, got.shape), *ref.bound(q, k, v, 0.0, out16=out16))


# ---- keys whose weight is zero ------------------------------------------------------------

# keys, heads, key heads: one part, a few, more than eight
FAR = [(300, 4, 2), (700, 4, 2), (2500, 4, 2), (8000, 2, 1)]


@pytest.mark.parametrize("S,H,Hkv", FAR)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("out16", [True, False])
def test_values_of_weightless_keys(ctx, S, H, Hkv, bad, out16):
    """a slope takes far keys' weights to zero: what their values hold does not reach the row, neither within the part
    that holds them nor where parts are joined, and a near one's does"""
    print(f"weightless {S} {bad} {out16}", flush=True)
    rng = np.random.default_rng(S)
    q, k, v = qkv(rng, 1, 3, S, H, Hkv, 48)
    v[0, 0], v[0, 5, 0, 3], v[0, 50:S - 150:50, :, 7] = bad, bad, bad
    slopes = np.full(H, 8.0, F32)
    got = check_masked(ctx, q, k, v, out16=out16, causal=True, slopes=slopes)
    assert np.isfinite(got.astype(F64)).all()
    v[0, S - 3, 0, 9] = bad
    check_masked(ctx, q, k, v, out16=out16, causal=True, slopes=slopes)


@pytest.mark.parametrize("S,spare", [(240, 0), (700, 10), (2500, 900)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("out16", [True, False])
def test_cached_values_of_weightless_keys(ctx, S, spare, bad, out16):
    """the same over the cache, whole blocks that read as NaN among them, in one part, a few and many"""
    print(f"weightless cached {S} {spare} {bad} {out16}", flush=True)
    rng = np.random.default_rng(S + spare)
    H, Hkv, D = 4, 2, 48
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, [S - 3], [3], H, Hkv, D, spare=spare)
        v[0, 0], v[0, 5, 0, 3], v[0, 50:S - 170:50, :, 7] = bad, bad, bad
        c.append(k[:, :S], v[:, :S], [0])
        got = check_cache(c, q, k, v, [S - 3], [3], have, out16=out16, slopes=np.full(H, 8.0, F32))
        assert np.isfinite(got.astype(F64)).all()


def test_prefixes_of_any_number(ctx):
    """a prefix below zero is none, one past the keys is all of them"""
    rng = np.random.default_rng(7)
    q, k, v = qkv(rng, 5, 30, 70, 2, 1, 32)
    check_masked(ctx, q, k, v, causal=True, prefix=np.array([-2 ** 31, -1, 0, 2 ** 31 - 1, 71], I32))


# ---- sequences that a call refuses, in parts ----------------------------------------------


@pytest.mark.parametrize("spare", [10, 900])
@pytest.mark.parametrize("S", [1, 4])
def test_cache_refuses_bad_numbers_in_parts(ctx, spare, S):
    """refused, ragged and good sequences, and pages outside the pool in an early and in a late part"""
    print(f"refused in parts {spare} {S}", flush=True)
    rng = np.random.default_rng(spare + S)
    H, Hkv, D = 4, 2, 48
    lens, new = [1500, 1500, 1200, 40, 900, 7], [S, S, S, max(S - 2, 0), S, S]
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, lens, new, H, Hkv, D, spare=spare)
        for out16 in (True, False):
            want = check_cache(c, q, k, v, lens, new, have, out16=out16)
            before = c.state()
            good = c.table
            table = good.copy()
            table[0, 45], table[1, 0], table[2, 20], table[4, 29:], table[3, 2:] = c.pages, -1, -2 ** 31, -7, -7
            c.set_table(table)
            got = c.attend(q, lens, new, out16=out16)
            # sequence 4's last whole block is number 27, sequence 3's 0: what lies behind is not read
            assert np.isnan(got[:3]).all() and np.array_equal(got[3:], want[3:])
            c.set_table(good)
            bad = [lens[0], -1, 32 * c.nb, lens[3], 2 ** 31 - 1, lens[5]]
            n = [S + 1, S, S, new[3], S, -1]
            for cap in (0.0, 9.0):
                got = c.attend(q, bad, n, out16=out16, cap=cap)
                assert np.isnan(got[[0, 1, 2, 4, 5]]).all()
                assert (got[3, new[3]:] == 7).all() and np.isfinite(got[3].astype(F64)).all()
            assert np.array_equal(c.attend(q, bad, n, out16=out16)[3], want[3])
            c.append(k[:, :S], v[:, :S], bad, [n[0], n[1], n[2], 0, n[4], n[5]])
            for x, y in zip(c.state(), before):
                assert np.array_equal(x, y, equal_nan=x.dtype != np.uint8)


# ---- together -----------------------------------------------------------------------------


def test_drafted_tokens_are_taken_back(ctx):
    """a prompt, then drafted tokens of which some are kept, again and again, eager and replayed: the cache and the
    rows are those of the tokens kept"""
    rng = np.random.default_rng(9)
    B, H, Hkv, D, S, P = 2, 4, 2, 48, 5, 37
    n = 150
    k, v = tokens(rng, B, n, Hkv, D)
    with Dev(ctx) as dev:
        c = Cache(dev, B, Hkv, D, 6, rng)
        c.append(k[:, :P], v[:, :P], [0, 0])
        have = np.array([P, P])
        lens = dev.up(have, I32)
        dk, dv, dq = (dev.up(np.zeros((B, S, h, D), F16)) for h in (Hkv, Hkv, H))
        o, st, kst = dev.up(np.zeros((B, S, H, D), F32)), (1, H * D, D, S * H * D), (1, Hkv * D, D, S * Hkv * D)

        def step():
            ctx.kv8_append(c.h, dk, dv, kst, S, lens)
            ctx.kv8_attn(c.h, dq, st, S, lens, None, H, 0.2, o=o, o_strides=st)

        graph = None
        for t in range(18):
            keep = rng.integers(0, S + 1, B)
            rows = [np.stack([x[b, have[b]:have[b] + S] for b in range(B)]) for x in (k, v)]
            for x in rows:                                                # the tokens not kept are other ones
                for b in range(B):
                    x[b, keep[b]:] = rng.standard_normal((S - keep[b], Hkv, D))
            q = rng.standard_normal((B, S, H, D)).astype(F16)
            for d, x in ((dk, rows[0]), (dv, rows[1]), (dq, q)):
                ctx.write(d, x)
            if t == 1:
                ctx.graph_begin()
                step()
                graph = ctx.graph_end()
            graph.launch() if graph else step()
            got = dev.get(o, (B, S, H, D), F32)
            for b in range(B):
                kk = np.concatenate([k[b, :have[b]], rows[0][b]])
                vv = np.concatenate([v[b, :have[b]], rows[1][b]])
                kk, vv, m = ref.cache_values(kk), ref.cache_values(vv), have[b] + S
                tol, rel = ref.bound(q[b:b + 1], kk[None], vv[None], 0.2)
                for i in range(S):
                    for h in range(H):
                        want = ref.attention_row(q[b, i, h].astype(F64), kk[:, h // 2], vv[:, h // 2], 0.2, 0.0, None, have[b] + i,
                                                 np.arange(m) <= have[b] + i)
                        close(got[b, i, h], want, tol, rel)
            ctx.kv8_advance(lens, dev.up(keep, I32), B, S)
            have = have + keep
        assert dev.get(lens, B, I32).tolist() == have.tolist()
        rk, rv = c.read(have, n)
        for b in range(B):
            for got, x in ((rk, k), (rv, v)):
                assert np.array_equal(got[b, :, :have[b]], ref.cache_values(x[b, :have[b]]).astype(F32).transpose(1, 0, 2))
        graph.destroy()


@pytest.mark.parametrize("spare", [1, 10, 900])
def test_a_sequence_does_not_depend_on_the_others(ctx, spare):
    """the same bits at another place of a batch of the same shape, beside sequences of other lengths"""
    rng = np.random.default_rng(spare)
    H, Hkv, D, S = 4, 2, 48, 3
    lens, new = np.array([700, 40, 1200]), np.array([3, 1, 2])
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, list(lens), list(new), H, Hkv, D, spare=spare)
        for kw in ({}, {"cap": 9.0, "slopes": np.full(H, 0.05, F32)}):
            for out16 in (True, False):
                want = c.attend(q, lens, new, out16=out16, **kw)
                at = np.array([2, 0, 1])
                tails = (c.kt, c.vt)
                one = [dev.get(x, c.B * Hkv * 64 * D, F16).reshape(c.B, -1)[at] for x in tails]
                c.kt, c.vt = dev.up(one[0]), dev.up(one[1])
                c.set_table(c.table[at])
                got = c.attend(q[at], lens[at], new[at], out16=out16, **kw)
                assert np.array_equal(got, want[at])
                short = lens[at].copy()
                short[0], short[2] = 0, 7                                 # (their own rows are other ones)
                got = c.attend(q[at], short, new[at], out16=out16, **kw)
                assert np.array_equal(got[1], want[at][1])
                c.kt, c.vt = tails
                c.set_table(c.table)
    q, k, v = qkv(rng, 3, 70, 300, H, Hkv, D)
    docs = np.sort(rng.integers(0, 4, (3, 300)).astype(I32), 1)
    want = run_masked(ctx, q, k, v, docs=docs, causal=True)
    at = np.array([1, 2, 0])
    assert np.array_equal(run_masked(ctx, q[at], k[at], v[at], docs=docs[at], causal=True), want[at])
    docs[1:] = 0
    assert np.array_equal(run_masked(ctx, q, k, v, docs=docs, causal=True)[0], want[0])
