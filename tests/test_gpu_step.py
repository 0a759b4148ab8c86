"""GPU parity of what a generating step does beside attention under masks: rotary positions, appending with the rotation on
the way, attention over shared blocks and sampling, each against its definition in 64 bits (tests/step_oracle.py and
tests/gen_oracle.py, which derive the tolerances)."""
import numpy as np
import pytest

import edge_maskgit_amd as ema
from tests import gen_oracle as gen
from tests import step_oracle as ref
from tests.test_gpu_generate import Cache, Dev, cache_case, close, ctx, tokens  # noqa: F401

pytestmark = pytest.mark.gpu
F16, F32, F64, I32 = np.float16, np.float32, np.float64, np.int32


def freqs_of(pairs):
    return [10000.0 ** (-i / max(n, 1)) for n in pairs for i in range(n)]


def positions(rng, axes, B, S, far=100):
    return rng.integers(-3, far, (axes, B, S)).astype(I32)


# ---- rotary positions -------------------------------------------------------------------------


def run_rope(ctx, x, pos, pairs, freqs, order, out16, first=None, new=None, fill=7.0):
    """contiguous [B,S,H,D] rows; pos [axes,B,S] or None"""
    B, S, H, D = x.shape
    st = (1, H * D, D, S * H * D)
    with Dev(ctx) as dev:
        y = dev.up(np.full(x.shape, fill, F16 if out16 else F32))
        rot = ema.Rope(pairs, freqs, order, dev.up(pos), (1, S, B * S))
        ctx.rope(rot, dev.up(x), st, D, S, H, B, in16=x.dtype == F16, first=dev.up(first, I32), new=dev.up(new, I32), y_strides=st,
                 **{"y16" if out16 else "y": y})
        return dev.get(y, x.shape, F16 if out16 else F32)


def check_rope(got, x, pos, pairs, freqs, order, out16):
    want = ref.rope(x, pos, pairs, freqs, order)
    over = np.abs(got.astype(F64) - want) - ref.rope_bound(x, pairs, order, out16)
    assert over.max() <= 0, f"past the bound by {over.max():.3g}"
    rest = 2 * sum(pairs)
    assert np.array_equal(got[..., rest:], x[..., rest:].astype(got.dtype))


# B, S, H, D, pairs of each axis: granules of 8, 4 and 1 pairs, whole and part of a head, odd numbers of everything
ROPES = [(1, 1, 1, 2, [1]), (2, 3, 1, 16, [8]), (1, 257, 32, 48, [12, 12]), (3, 17, 5, 64, [16]), (2, 33, 7, 128, [16, 24, 24]), (1, 70, 3, 80, [5, 7, 9, 11]),
         (1, 9, 40, 128, [64]), (2, 5, 3, 96, [8, 0, 16]), (1, 6, 2, 30, [7, 8]), (5, 2, 9, 112, [0]), (1, 1000, 2, 6, [2, 1]), (1, 3, 70, 72, [36])]


@pytest.mark.parametrize("order", [0, 1, 2])
@pytest.mark.parametrize("shape", ROPES)
def test_rope(ctx, shape, order):
    print(f"rope {shape} {order}", flush=True)
    B, S, H, D, pairs = shape
    rng = np.random.default_rng(B + S + D)
    x = rng.standard_normal((B, S, H, D)) * 3
    pos = positions(rng, len(pairs), B, S)
    f = freqs_of(pairs)
    for t in (F16, F32):
        for out16 in (False, True):
            check_rope(run_rope(ctx, x.astype(t), pos, pairs, f, order, out16), x.astype(t), pos, pairs, f, order, out16)


@pytest.mark.parametrize("order", [0, 1, 2])
def test_rope_many_rows(ctx, order):
    """several heads of a thread, in steps that do not divide the heads"""
    rng = np.random.default_rng(order)
    for B, S, H, D, pairs in ((2, 3000, 37, 64, [16, 16]), (1, 4097, 21, 48, [12, 12]), (1, 9000, 9, 32, [5])):
        x = rng.standard_normal((B, S, H, D)).astype(F16)
        pos, f = positions(rng, len(pairs), B, S, 5000), freqs_of(pairs)
        check_rope(run_rope(ctx, x, pos, pairs, f, order, True), x, pos, pairs, f, order, True)
        check_rope(run_rope(ctx, x, pos, pairs, f, order, False), x, pos, pairs, f, order, False)


def test_rope_far_positions(ctx):
    """angles of positions to the ends of 32 bits, of any frequency to 16 and of either sign: whole turns leave no error"""
    rng = np.random.default_rng(5)
    pos = np.array([0, 1, -1, 100003, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 123456789, -987654321], I32).reshape(1, 1, -1)
    f = [1.0, -1.0, 16.0, -16.0, 1e-4, 2 * np.pi, np.pi / 2, 1e-9, 0.0, 3.7, 0.1, np.pi, 1 / 3, 15.99999, -1e-3, 5.0]
    x = rng.standard_normal((1, 9, 2, 32)).astype(F32)
    check_rope(run_rope(ctx, x, pos, [16], f, 0, False), x, pos, [16], f, 0, False)


def test_rope_consecutive_positions(ctx):
    rng = np.random.default_rng(6)
    pairs, f = [6, 10], freqs_of([6, 10])
    x = rng.standard_normal((3, 40, 2, 32)).astype(F32)
    first = np.array([0, 1000000, -20], I32)
    run = np.broadcast_to((first[:, None] + np.arange(40))[None], (2, 3, 40))
    check_rope(run_rope(ctx, x, None, pairs, f, 2, False, first=first), x, run, pairs, f, 2, False)
    zero = np.broadcast_to(np.arange(40)[None, None], (2, 3, 40))
    check_rope(run_rope(ctx, x, None, pairs, f, 1, False), x, zero, pairs, f, 1, False)


def test_rope_leaves_other_rows_alone(ctx):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((5, 6, 2, 16)).astype(F16)
    x[0, 3:] = np.nan
    pos = positions(rng, 1, 5, 6)
    new = [3, 0, 6, -1, 7]                                  # the last two do not fit
    for out16 in (False, True):
        got = run_rope(ctx, x, pos, [8], freqs_of([8]), 0, out16, new=new)
        assert (got[0, 3:] == 7).all() and (got[[1, 3, 4]] == 7).all()
        check_rope(got[:1, :3], x[:1, :3], pos[:, :1, :3], [8], freqs_of([8]), 0, out16)
        check_rope(got[2:3], x[2:3], pos[:, 2:3], [8], freqs_of([8]), 0, out16)


def test_rope_layouts(ctx):
    """views of fused rows, heads outside the tokens, features apart, odd offsets, one row of positions for all, in place: what
    contiguous rows give"""
    rng = np.random.default_rng(8)
    B, S, H, D, pairs = 2, 19, 4, 32, [4, 8]
    f = freqs_of(pairs)
    for t in (F16, F32):
        x = rng.standard_normal((B, S, H, D)).astype(t)
        one = np.repeat(positions(rng, 2, 1, S), B, 1)
        for order in (0, 1, 2):
            want = run_rope(ctx, x, one, pairs, f, order, t == F16)
            out = "y16" if t == F16 else "y"
            for pad in (0, 8, 4, 3):
                rows = np.full((B, S, H * D + pad), 5, t)
                rows[..., :H * D] = x.reshape(B, S, -1)
                with Dev(ctx) as dev:
                    d, st = dev.up(rows), (1, H * D + pad, D, S * (H * D + pad))
                    rot = ema.Rope(pairs, f, order, dev.up(one[:, :1]), (1, 0, S))
                    ctx.rope(rot, d, st, D, S, H, B, in16=t == F16, **{out: d})
                    got = dev.get(d, rows.shape, t)
                    assert np.array_equal(got[..., :H * D].reshape(x.shape), want) and (got[..., H * D:] == 5).all(), (pad, order)
            with Dev(ctx) as dev:                           # features outermost, an odd offset; heads outside the tokens behind it
                e = np.dtype(t).itemsize
                d = dev.up(np.r_[t(0), np.ascontiguousarray(x.transpose(3, 0, 2, 1)).ravel()])
                y = dev.up(np.zeros((B, H, S, D), t))
                ctx.rope(ema.Rope(pairs, f, order, dev.up(one), (1, S, B * S)), d.ptr + e, (B * H * S, 1, S, H * S), D, S, H, B,
                         in16=t == F16, y_strides=(1, D, S * D, H * S * D), **{out: y})
                assert np.array_equal(dev.get(y, (B, H, S, D), t).transpose(0, 2, 1, 3), want)


@pytest.mark.parametrize("B,S,H,D,pairs", [(2, 100, 16, 48, [24]), (1, 1000, 32, 64, [16, 16]), (3, 37, 5, 32, [4, 8])])
@pytest.mark.parametrize("t", [F16, F32])
def test_rope_rows_of_every_alignment(ctx, B, S, H, D, pairs, t):
    """rows, heads and pointers at multiples of one, two, three, four and six elements, of x, of y and in place: what contiguous
    rows give, every token of it, and nothing beside it"""
    print(f"rope alignment {B} {S} {H} {D} {pairs} {t.__name__}", flush=True)
    rng = np.random.default_rng(D)
    f, n, e = freqs_of(pairs), H * D, np.dtype(t).itemsize
    x = rng.standard_normal((B, S, H, D)).astype(t)
    x[x == 9] = 8
    pos = positions(rng, len(pairs), B, S)
    out = "y16" if t == F16 else "y"
    for order in (0, 1, 2):
        want = run_rope(ctx, x, pos, pairs, f, order, t == F16)
        with Dev(ctx) as dev:
            rot = ema.Rope(pairs, f, order, dev.up(pos), (1, S, B * S))
            dx, st = dev.up(x), (1, n, D, S * n)
            for pad, gap, off in ((2, 0, 0), (6, 0, 0), (0, 2, 0), (0, 6, 0), (0, 0, 2), (0, 0, 6), (2, 2, 2), (0, 0, 4), (0, 0, 1), (1, 0, 0), (3, 3, 3), (4, 4, 0), (8, 8, 8)):
                w = H * (D + gap) + pad                             # rows of heads D + gap apart, from element `off` on
                rows = np.full(off + B * S * w, 9, t)
                rows[off:].reshape(B, S, w)[..., :H * (D + gap)].reshape(B, S, H, D + gap)[..., :D] = x
                there = np.zeros(rows.shape, bool)
                there[off:].reshape(B, S, w)[..., :H * (D + gap)].reshape(B, S, H, D + gap)[..., :D] = True
                wide = (1, w, D + gap, S * w)
                d, y, z = dev.up(rows), dev.up(np.full(x.shape, 9, t)), dev.up(np.full(rows.shape, 9, t))
                ctx.rope(rot, d.ptr + e * off, wide, D, S, H, B, in16=t == F16, y_strides=st, **{out: y})
                ctx.rope(rot, dx, st, D, S, H, B, in16=t == F16, y_strides=wide, **{out: z.ptr + e * off})
                ctx.rope(rot, d.ptr + e * off, wide, D, S, H, B, in16=t == F16, **{out: d.ptr + e * off})
                assert np.array_equal(dev.get(y, x.shape, t), want), (order, pad, gap, off)
                for b in (z, d):
                    got = dev.get(b, rows.shape, t)
                    assert np.array_equal(got[there], want.ravel()) and (got[~there] == 9).all(), (order, pad, gap, off)


def test_rope_of_anything(ctx):
    """infinities and NaN stay within their pair"""
    x = np.ones((1, 4, 1, 16), F32)
    x[0, 1, 0, 3], x[0, 2, 0, 5], x[0, 3, 0, 15] = np.nan, np.inf, -np.inf
    pos = np.arange(4, dtype=I32).reshape(1, 1, 4)
    got = run_rope(ctx, x, pos, [8], freqs_of([8]), 0, False)[0, :, 0]
    bad = ~np.isfinite(got)
    assert sorted(zip(*np.nonzero(bad))) == [(1, 3), (1, 11), (2, 5), (2, 13), (3, 7), (3, 15)]


def test_rope_offsets_past_32_bits(ctx):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((2, 3, 2, 32)).astype(F16)
    pos, f = positions(rng, 1, 2, 3), freqs_of([16])
    want = run_rope(ctx, x, pos, [16], f, 0, True)
    token, seq = (1 << 29) + 64, 3 * (1 << 29) + 4096                 # a GiB and more between rows
    with Dev(ctx) as dev:
        big = ctx.alloc(2 * (2 * seq + (1 << 16)))
        dev.bufs.append(big)
        for b in range(2):
            for i in range(3):
                r = np.ascontiguousarray(x[b, i])
                ctx._check(ema.lib().mgh_h2d(ctx.h, big.ptr + 2 * (b * seq + i * token), r.ctypes.data, r.nbytes))
        y = dev.up(np.zeros_like(x))
        ctx.rope(ema.Rope([16], f, 0, dev.up(pos), (1, 3, 6)), big, (1, token, 32, seq), 32, 3, 2, 2, y16=y, y_strides=(1, 64, 32, 192))
        assert np.array_equal(dev.get(y, x.shape, F16), want)


# ---- appending with the rotation on the way ------------------------------------------------------


def append_rope(c, rot, k, v, q, lens, new=None, in16=True, fill=7.0):
    """k, v [B,S,Hkv,D], q [B,S,H,D] -> the rotated queries"""
    B, S, H, D = q.shape
    w, t = c.Hkv * D, F16 if in16 else F32
    out = c.dev.up(np.full(q.shape, fill, F16))
    st = (1, H * D, D, S * H * D)
    c.dev.ctx.kv8_append_rope(c.h, rot, c.dev.up(k, t), c.dev.up(v, t), (1, w, D, S * w), S, c.dev.up(lens, I32), c.dev.up(new, I32),
                              in16=in16, q=c.dev.up(q, t), q_strides=st, H=H, q_out=out, qo_strides=st)
    return c.dev.get(out, q.shape, F16)


def same_state(a, b):
    for x, y in zip(a, b):
        assert np.array_equal(x, y, equal_nan=x.dtype != np.uint8)


@pytest.mark.parametrize("order", [0, 1, 2])
@pytest.mark.parametrize("D,Hkv,G,pairs", [(16, 1, 1, [8]), (48, 3, 1, [12, 12]), (64, 2, 4, [16]), (80, 1, 2, [5, 7, 9]), (128, 2, 3, [16, 24, 24]), (96, 2, 1, [0])])
def test_rotated_append_is_rope_and_append(ctx, D, Hkv, G, pairs, order):
    """the same cache, byte for byte, as appending keys that were rotated in 64 bits and rounded once (the kernel's own 64 bits
    are off by 2^-45: one value in 2^33 lies so near a border of fp16's), and mgh_rope's queries; in odd pieces, from either
    type, positions given and not"""
    print(f"append {D} {Hkv} {pairs} {order}", flush=True)
    rng = np.random.default_rng(D + order)
    B, n, H = 2, 150, Hkv * G
    k, v = tokens(rng, B, n, Hkv, D)
    q = rng.standard_normal((B, n, H, D)).astype(F16)
    f = freqs_of(pairs)
    pos = positions(rng, len(pairs), B, n)
    for in16 in (True, False):
        t = F16 if in16 else F32
        for given in (True, False):
            at = pos if given else np.broadcast_to(np.arange(n, dtype=I32), (len(pairs), B, n))
            with Dev(ctx) as dev:
                tq = run_rope(ctx, q.astype(t), at, pairs, f, order, True)
                turned = ref.rope(k, at, pairs, f, order).astype(F16)
                want = Cache(dev, B, Hkv, D, 5, np.random.default_rng(1))
                want.append(turned, v, [0, 0])
                for steps in ([np.array([n, n])], [np.array([7, 33])] * 22, [np.array([0, 64]), np.array([90, 1])] * 10):
                    c, done = Cache(dev, B, Hkv, D, 5, np.random.default_rng(1)), np.zeros(B, int)
                    for new in steps:
                        new = np.minimum(new, n - done)
                        S = max(int(new.max()), 1)
                        kk, vv, qq = np.full((B, S, Hkv, D), np.nan, F16), np.full((B, S, Hkv, D), np.nan, F16), np.full((B, S, H, D), np.nan, F16)
                        pp = np.zeros((len(pairs), B, S), I32)
                        for b in range(B):
                            s = slice(done[b], done[b] + new[b])
                            kk[b, :new[b]], vv[b, :new[b]], qq[b, :new[b]] = k[b, s], v[b, s], q[b, s]
                            pp[:, b, :new[b]] = pos[:, b, s]
                        rot = ema.Rope(pairs, f, order, dev.up(pp) if given else None, (1, S, B * S))
                        got = append_rope(c, rot, kk, vv, qq, done, new, in16)
                        for b in range(B):
                            assert np.array_equal(got[b, :new[b]], tq[b, done[b]:done[b] + new[b]])
                            assert (got[b, new[b]:] == 7).all()             # rows past a sequence's tokens: as they were
                        done = done + new
                    assert (done == n).all()
                    same_state(c.state(), want.state())


# (B, S, Hkv, G, D): threads for 8 waves per SIMD with 2, 4 and 8 heads of each, groups that these do not divide, and few rows
MANY = [(2, 2100, 8, 4, 128), (1, 2500, 8, 3, 128), (3, 900, 4, 17, 48), (2, 700, 2, 32, 128), (2, 33, 1, 9, 64), (1, 1, 2, 16, 128), (2, 2100, 16, 2, 80)]


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("B,S,Hkv,G,D", MANY)
def test_rotated_append_turns_every_query_head(ctx, B, S, Hkv, G, D, aligned):
    """mgh_rope's queries, all of them, where threads take several heads of a group, and nothing past them"""
    print(f"append heads {B} {S} {Hkv} {G} {D} {aligned}", flush=True)
    rng = np.random.default_rng(S + G)
    H, pairs = Hkv * G, [D // 2]
    f = freqs_of(pairs)
    q = rng.standard_normal((B, S, H, D)).astype(F16)
    q[q == 7] = 6
    k, v = tokens(rng, B, S, Hkv, D)
    at = np.broadcast_to(np.arange(S, dtype=I32), (1, B, S))
    w = H * D + (8 if aligned else 1)
    rows = np.full((B, S, w), 7, F16)
    rows[..., :H * D] = q.reshape(B, S, H * D)
    with Dev(ctx) as dev:
        want = run_rope(ctx, q, at, pairs, f, 0, True)
        c = Cache(dev, B, Hkv, D, (S + 31) // 32, np.random.default_rng(1))
        out, st, kst = dev.up(np.full(rows.shape, 7, F16)), (1, w, D, S * w), (1, Hkv * D, D, S * Hkv * D)
        c.dev.ctx.kv8_append_rope(c.h, ema.Rope(pairs, f, 0), dev.up(k, F16), dev.up(v, F16), kst, S, dev.up(np.zeros(B, I32)), None,
                                  in16=True, q=dev.up(rows), q_strides=st, H=H, q_out=out, qo_strides=st)
        got = dev.get(out, rows.shape, F16)
    assert np.array_equal(got[..., :H * D].reshape(q.shape), want)
    assert (got[..., H * D:] == 7).all()


def test_rotated_append_against_the_definition(ctx):
    """keys rotated in 64 bits and rounded once; codes of whole blocks from exactly the fp16 values that the ring had"""
    rng = np.random.default_rng(3)
    D, Hkv, pairs = 64, 2, [16, 16]
    f = freqs_of(pairs)
    k, v = tokens(rng, 1, 50, Hkv, D)
    q = np.zeros((1, 50, Hkv, D), F16)
    pos = positions(rng, 2, 1, 50, 1000)
    with Dev(ctx) as dev:
        c = Cache(dev, 1, Hkv, D, 2, rng)
        rot = lambda a, b: ema.Rope(pairs, f, 0, dev.up(np.ascontiguousarray(pos[:, :, a:b])), (1, b - a, b - a))  # noqa: E731
        append_rope(c, rot(0, 31), k[:, :31], v[:, :31], q[:, :31], [0])
        early, _ = c.read([31], 31)
        turned = ref.rope(k, pos, pairs, f, 0).astype(F16)
        assert np.array_equal(turned[0, :31], early[0].transpose(1, 0, 2))
        append_rope(c, rot(31, 50), k[:, 31:], v[:, 31:], q[:, 31:], [31])
        got, gv = c.read([50], 50)
        assert np.array_equal(got[0], gen.cache_values(turned[0]).astype(F32).transpose(1, 0, 2))
        assert np.array_equal(gv[0], gen.cache_values(v[0]).astype(F32).transpose(1, 0, 2))


def test_rotated_append_of_any_size(ctx):
    """fp32 keys from fp16's smallest numbers to past its largest, at positions to the ends of 32 bits: rounded once"""
    rng = np.random.default_rng(33)
    D, Hkv, pairs = 32, 2, [16]
    f = [1.0, -1.0, 16.0, 1e-4, 2 * np.pi, np.pi / 2, 1e-9, 0.0, 3.7, 0.1, np.pi, 1 / 3, 15.99999, -1e-3, 5.0, 0.7]
    size = 2.0 ** rng.integers(-30, 17, (1, 30, Hkv, D))
    size[:, 20:] = 2.0 ** rng.integers(-149, -100, (1, 10, Hkv, D))         # (products below fp32's smallest number)
    k = (rng.standard_normal((1, 30, Hkv, D)) * size).astype(F32)
    k[0, 3, 0, 2], k[0, 4, 1, 7], k[0, 5, 0, 31] = np.inf, np.nan, -np.inf
    pos = rng.integers(-2 ** 31, 2 ** 31, (1, 1, 30)).astype(I32)
    pos[0, 0, :4] = 0, -2 ** 31, 2 ** 31 - 1, 5
    for order in (0, 1):
        with Dev(ctx) as dev:
            c = Cache(dev, 1, Hkv, D, 1, rng)
            append_rope(c, ema.Rope(pairs, f, order, dev.up(pos), (1, 30, 30)), k, k, np.zeros((1, 30, Hkv, D), F32), [0], in16=False)
            got = dev.get(c.kt, (1, Hkv, 64, D), F16)[0, :, :30].transpose(1, 0, 2)
        with np.errstate(all="ignore"):
            want = ref.rope(k, pos, pairs, f, order)[0]
            # the frequency is a whole number of 2^-64 turns: an angle at 2^31 is off by 2^-33 turns, 7e-10 of |a| + |b|
            room = ref.rope_bound(k, pairs, order, False)[0] / (5 * ref.U) * 1e-9
            lo, hi = (want - room).astype(F16), (want + room).astype(F16)
        odd = ~np.isfinite(want)
        assert not np.isfinite(got[odd]).any()
        assert ((got >= lo) & (got <= hi))[~odd].all()


def test_rotated_append_refuses_bad_numbers_on_the_device(ctx):
    rng = np.random.default_rng(4)
    B, Hkv, D = 4, 1, 32
    k, v = tokens(rng, B, 70, Hkv, D)
    q = rng.standard_normal((B, 1, 2, D)).astype(F16)
    rot = ema.Rope([16], freqs_of([16]))
    with Dev(ctx) as dev:
        c = Cache(dev, B, Hkv, D, 3, rng)
        c.append(k, v, [0] * B)
        before = c.state()
        got = append_rope(c, rot, k[:, :1], v[:, :1], q, [-1, 96, 70, 70], [1, 1, 2, -1])
        assert (got == 7).all()
        same_state(c.state(), before)
        table = c.table.copy()
        table[0, 2], table[1, 2] = c.pages, -5                  # the block that the call completes
        c.set_table(table)
        append_rope(c, rot, np.repeat(k[:, :1], 26, 1), np.repeat(v[:, :1], 26, 1), np.repeat(q, 26, 1), [70] * B, [26, 26, 26, 26])
        gk, gs = c.state()[0].reshape(c.pages, -1), c.state()[2].reshape(c.pages, -1)
        for p in set(range(c.pages)) - set(table.ravel().tolist()):
            assert (gk[p] == before[0].reshape(c.pages, -1)[p]).all() and np.array_equal(gs[p], before[2].reshape(c.pages, -1)[p], equal_nan=True)


def test_rotated_append_layouts(ctx):
    """fused rows with odd gaps, queries in place, features apart, keys alone"""
    rng = np.random.default_rng(5)
    B, S, H, Hkv, D, pairs = 2, 40, 4, 2, 48, [12, 12]
    f, w = freqs_of(pairs), (H + 2 * Hkv) * D
    q, k, v = (rng.standard_normal((B, S, n, D)).astype(F16) for n in (H, Hkv, Hkv))
    pos = positions(rng, 2, B, S)
    for order in (0, 1, 2):
        with Dev(ctx) as dev:
            rot = ema.Rope(pairs, f, order, dev.up(pos), (1, S, B * S))
            fresh = lambda: Cache(dev, B, Hkv, D, 2, np.random.default_rng(2))  # noqa: E731
            one = fresh()
            want = append_rope(one, rot, k, v, q, [5, 0])
            for pad in (0, 8, 4, 1):
                rows = np.full((B, S, w + pad), 3, F16)
                rows[..., :w] = np.concatenate([x.reshape(B, S, -1) for x in (q, k, v)], 2)
                c, d = fresh(), dev.up(rows)
                st = (1, w + pad, D, S * (w + pad))
                ctx.kv8_append_rope(c.h, rot, d.ptr + 2 * H * D, d.ptr + 2 * (H + Hkv) * D, st, S, dev.up([5, 0], I32), q=d, q_strides=st, H=H,
                                    q_out=d, qo_strides=st)
                same_state(c.state(), one.state())
                got = dev.get(d, rows.shape, F16)
                assert np.array_equal(got[..., :H * D].reshape(q.shape), want) and np.array_equal(got[..., H * D:], rows[..., H * D:])
            c = fresh()
            ks, vs = (dev.up(np.ascontiguousarray(x.transpose(3, 0, 2, 1))) for x in (k, v))
            ctx.kv8_append_rope(c.h, rot, ks, vs, (B * Hkv * S, 1, S, Hkv * S), S, dev.up([5, 0], I32))
            same_state(c.state(), one.state())


# ---- attention over shared blocks -----------------------------------------------------------------


def shared_case(dev, rng, group, shared, own, new, H, Hkv, D, spare=1):
    """sequences whose first shared[g] blocks are the same pages; own: tokens of each behind them, before the new ones"""
    B, S = len(own), max(max(new), 1)
    sh = [shared[b // group] for b in range(B)]
    lens = [32 * s + n for s, n in zip(sh, own)]
    c, q, k, v, have = cache_case(dev, rng, lens, new, H, Hkv, D, spare)
    table = c.table.copy()
    for b in range(B):
        first = b // group * group
        n = 32 * sh[b]
        k[b, :n], v[b, :n] = k[first, :n], v[first, :n]
        table[b, :sh[b]] = table[first, :sh[b]]
    c.set_table(table)
    c.append(k[:, :max(have)], v[:, :max(have)], [0] * B, have)
    return c, q, k, v, lens, have, table


def attend(c, q, lens, new, group, shared, most=None, in16=True, out16=True, cap=0.0, slopes=None, scale=None, fill=7.0):
    _, S, H, D = q.shape
    st = (1, H * D, D, S * H * D)
    o = c.dev.up(np.full(q.shape, fill, F16 if out16 else F32))
    c.dev.ctx.kv8_attn_shared(c.h, c.dev.up(q, F16 if in16 else F32), st, S, c.dev.up(lens, I32), c.dev.up(new, I32), group,
                              c.dev.up(shared, I32), max(shared) if most is None else most, H, D ** -0.5 if scale is None else scale,
                              in16=in16, cap=cap, slopes=c.dev.up(slopes, F32), o_strides=st, **{"o16" if out16 else "o": o})
    return c.dev.get(o, q.shape, F16 if out16 else F32)


def lost_weights(q, k, v, scale, cap, slope, p, seen):
    """what row_tolerance leaves out where the largest weight's own value is small: weights relative to the reference are at
    least 2^7 at the row's largest (the reference is set 7 below a score and later scores lie above it or below), and the
    low part of hi + lo is a multiple of 2^-24 there, so each weight may be off by 2^-25, 2^-32 of the largest, whatever its
    own size: it moves the output by that of |v_j - o|"""
    at = np.nonzero(seen)[0]
    s = (k[at] @ q) * scale
    s = cap * np.tanh(s / cap) if cap else s
    s = s if slope is None else s - slope * np.abs(p - at)
    w = np.exp(s - s.max())
    w = w / w.sum()
    return 2.0 ** -32 * w.max() * np.abs(v[at] - w @ v[at]).sum(0)


def check_rows(got, c, q, k, v, lens, new, have, out16, some=None, **kw):
    H, D = q.shape[2:]
    worst = 0
    for b in range(len(q)):
        kk, vv = gen.cache_values(k[b, :have[b]]), gen.cache_values(v[b, :have[b]])
        for i in range(new[b]):
            for h in range(H):
                if some is not None and (b, i, h) not in some:
                    continue
                g, p, sl = h // (H // c.Hkv), lens[b] + i, kw.get("slopes")
                args = (q[b, i, h].astype(F64), kk[:, g], vv[:, g], kw.get("scale") or D ** -0.5, kw.get("cap", 0.0),
                        None if sl is None else float(sl[h]), p, np.arange(have[b]) <= p)
                tol = gen.row_tolerance(*args, out16=out16) + (0 if out16 else 1.01 * lost_weights(*args))
                over = (np.abs(got[b, i, h].astype(F64) - gen.attention_row(*args)) / tol).max()
                worst = max(worst, over)
                assert over <= 1, ((b, i, h), over)
        assert (got[b, new[b]:] == 7).all()                                 # rows past a sequence's tokens: as they were
    return worst


# group, shared blocks of each group, own tokens and new tokens of each sequence, H, Hkv, D
SHARED = [(1, [1], [0], [1], 1, 1, 16), (3, [2], [0, 5, 40], [1, 1, 1], 4, 2, 32), (2, [3, 1, 0], [31, 0, 70, 64, 3], [1, 1, 1, 1, 1], 6, 2, 48),
          (4, [9], [100, 0, 1, 33], [5, 2, 0, 4], 4, 4, 48), (8, [20], [3, 0, 60, 7, 31, 32, 33, 1], [1] * 8, 8, 1, 64), (2, [40, 70], [10, 0, 90, 5], [2, 1, 3, 3], 4, 1, 128),
          (5, [0], [3, 0, 100, 64, 7], [1] * 5, 2, 1, 80), (3, [17, 5], [1, 2, 3, 4, 5], [3, 3, 1, 2, 3], 8, 2, 112), (20, [11], [0] * 20, [1] * 20, 8, 2, 96),
          (7, [33], [9] * 7, [6, 0, 6, 6, 1, 6, 6], 12, 1, 64)]


@pytest.mark.parametrize("kind", ["plain", "cap", "slopes"])
@pytest.mark.parametrize("case", SHARED)
def test_shared_attention(ctx, case, kind):
    print(f"shared {case} {kind}", flush=True)
    group, shared, own, new, H, Hkv, D = case
    rng = np.random.default_rng(sum(own) + D)
    kw = {"cap": {"cap": 3.0}, "slopes": {"slopes": (0.5 ** np.arange(1, H + 1)).astype(F32)}}.get(kind, {})
    with Dev(ctx) as dev:
        c, q, k, v, lens, have, _ = shared_case(dev, rng, group, shared, own, new, H, Hkv, D)
        for out16 in (True, False):
            got = attend(c, q, lens, new, group, shared, out16=out16, **kw)
            check_rows(got, c, q, k, v, lens, new, have, out16, **kw)
        check_rows(attend(c, q, lens, new, group, shared, most=c.nb, **kw), c, q, k, v, lens, new, have, True, **kw)


@pytest.mark.parametrize("group,shared,B,H,Hkv,D,new", [(64, [30], 64, 16, 4, 128, 1), (64, [70], 64, 8, 2, 64, 1), (33, [25, 12], 60, 4, 4, 48, 3), (16, [60, 3, 0, 41], 64, 8, 1, 32, 2)])
def test_shared_attention_many_rows(ctx, group, shared, B, H, Hkv, D, new):
    """tiles of rows of many sequences"""
    print(f"shared rows {group} {shared} {B} {H} {D} {new}", flush=True)
    rng = np.random.default_rng(D)
    own = rng.integers(0, 90, B).tolist()
    n = rng.integers(0, new + 1, B)
    n[0] = new
    n = n.tolist()
    with Dev(ctx) as dev:
        c, q, k, v, lens, have, _ = shared_case(dev, rng, group, shared, own, n, H, Hkv, D)
        rows = [(b, i, h) for b in range(B) for i in range(n[b]) for h in range(H)]
        some = {rows[i] for i in rng.permutation(len(rows))[:60]} | {rows[0], rows[-1]}
        for out16 in (True, False):
            for kw in ({}, {"cap": 4.0, "slopes": np.linspace(0, 0.1, H).astype(F32)}):
                got = attend(c, q, lens, n, group, shared, out16=out16, **kw)
                check_rows(got, c, q, k, v, lens, n, have, out16, some, **kw)
                assert np.isfinite(got).all()


def test_shared_attention_reads_the_first_row_of_the_table(ctx):
    """the other sequences' page numbers of shared blocks are not read; a bound past the groups' own changes nothing but bits"""
    rng = np.random.default_rng(11)
    group, shared, own, new = 3, [4, 6], [3, 50, 20, 1, 70], [1, 1, 1, 1, 1]
    with Dev(ctx) as dev:
        c, q, k, v, lens, have, table = shared_case(dev, rng, group, shared, own, new, 4, 2, 64)
        want = attend(c, q, lens, new, group, shared)
        bad = table.copy()
        for b in range(5):
            if b % group:
                bad[b, :shared[b // group]] = [-1, c.pages, 2 ** 31 - 1, -2 ** 31, 0, 1][:shared[b // group]]
        c.set_table(bad)
        assert np.array_equal(attend(c, q, lens, new, group, shared), want)
        check_rows(attend(c, q, lens, new, group, shared, most=c.nb), c, q, k, v, lens, new, have, True)


def test_shared_attention_refuses_bad_numbers_on_the_device(ctx):
    """a sequence shorter than what it shares, a group's number that does not fit, lengths that do not, pages outside the pool"""
    rng = np.random.default_rng(12)
    group, shared, own, new = 2, [3, 3, 3], [5, 9, 0, 40, 7, 8], [1] * 6
    with Dev(ctx) as dev:
        c, q, k, v, lens, have, table = shared_case(dev, rng, group, shared, own, new, 4, 2, 48)
        want = attend(c, q, lens, new, group, shared)
        check_rows(want, c, q, k, v, lens, new, have, True)
        short = list(lens)
        short[1], short[2] = 95, -1
        got = attend(c, q, short, new, group, shared)
        assert np.isnan(got[[1, 2]]).all() and np.array_equal(got[[0, 3, 4, 5]], want[[0, 3, 4, 5]])
        for n in (-1, 4, 2 ** 31 - 1):
            got = attend(c, q, lens, new, group, [3, n, 3], most=3)
            assert np.isnan(got[2:4]).all() and np.array_equal(got[[0, 1, 4, 5]], want[[0, 1, 4, 5]])
        got = attend(c, q, lens, [1, 2, 1, -1, 1, 0], group, shared)                # S is 1
        assert np.isnan(got[[1, 3]]).all() and np.array_equal(got[[0, 2, 4]], want[[0, 2, 4]]) and (got[5] == 7).all()
        lost = table.copy()
        lost[0, 1] = c.pages                                                       # a shared block of the first group
        lost[4, 3:], lost[3, 3] = -1, -9                                           # (sequence 4's open block is not read)
        c.set_table(lost)
        got = attend(c, q, lens, new, group, shared)
        assert np.isnan(got[[0, 1, 3]]).all() and np.array_equal(got[[2, 4, 5]], want[[2, 4, 5]])


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("out16", [True, False])
def test_shared_attention_of_anything(ctx, bad, out16):
    """a shared block of one head that holds an infinity or NaN reaches its rows of every sequence; one of a sequence's own
    reaches that sequence's"""
    rng = np.random.default_rng(13)
    group, shared, own, new, H, Hkv, D = 20, [6], [3] * 19 + [60], [1] * 20, 4, 2, 64
    with Dev(ctx) as dev:
        c, q, k, v, lens, have, _ = shared_case(dev, rng, group, shared, own, new, H, Hkv, D)
        k2, v2 = k.copy(), v.copy()
        v2[0, 70, 1, 5] = bad                                   # (sequence 0 writes the shared pages)
        v2[19, 32 * 6 + 3, 0, 9] = bad
        for b in range(1, 20):
            v2[b, :192] = v2[0, :192]
        c.append(k2[:, :max(have)], v2[:, :max(have)], [0] * 20, have)
        got = attend(c, q, lens, new, group, shared, out16=out16)
        assert np.isnan(got[:, :, 2:]).all() and np.isnan(got[19, :, :2]).all() and np.isfinite(got[:19, :, :2]).all()
        some = {(b, 0, h) for b in range(19) for h in (0, 1)}
        check_rows(got[:19], c, q[:19], k2[:19], np.where(np.isfinite(v2), v2, 0)[:19], lens[:19], new[:19], have[:19], out16, some)


def test_shared_attention_scores_of_any_size(ctx):
    """shared scores far above or far below the own ones, weights past fp16's range between the parts"""
    rng = np.random.default_rng(14)
    group, shared, own, new, H, Hkv, D = 12, [5], [20] * 12, [1] * 12, 4, 1, 32
    with Dev(ctx) as dev:
        c, q, k, v, lens, have, _ = shared_case(dev, rng, group, shared, own, new, H, Hkv, D)
        for lift in (6, -6):
            k2 = k.copy()
            k2[:, :160] += F16(lift)
            c.append(k2[:, :max(have)], v[:, :max(have)], [0] * 12, have)
            for scale in (1.0, 0.01, -1.0):
                for out16 in (True, False):
                    qq = np.abs(q)
                    got = attend(c, qq, lens, new, group, shared, out16=out16, scale=scale)
                    check_rows(got, c, qq, k2, v, lens, new, have, out16, scale=scale)


def test_shared_attention_queries_of_any_layout(ctx):
    rng = np.random.default_rng(15)
    group, shared, own, new, H, Hkv, D = 3, [4], [3, 30, 9], [2, 2, 2], 4, 2, 32
    with Dev(ctx) as dev:
        c, q, k, v, lens, have, _ = shared_case(dev, rng, group, shared, own, new, H, Hkv, D)
        want = attend(c, q, lens, new, group, shared)
        assert np.array_equal(attend(c, q.astype(F32), lens, new, group, shared, in16=False), want)
        x = dev.up(np.r_[F16(0), np.ascontiguousarray(q.transpose(3, 0, 2, 1)).ravel()])
        o = dev.up(np.zeros((3, H, 2, D), F16))
        ctx.kv8_attn_shared(c.h, x.ptr + 2, (3 * H * 2, 1, 2, H * 2), 2, dev.up(lens, I32), None, 3, dev.up(shared, I32), 4, H, D ** -0.5, o16=o)
        assert np.array_equal(dev.get(o, (3, H, 2, D), F16).transpose(0, 2, 1, 3), want)


# ---- sampling -----------------------------------------------------------------------------


def run_sample(ctx, x, u, one_row=False, pad=0, **kw):
    rows, V = (len(u), x.shape[-1])
    with Dev(ctx) as dev:
        arr = {n: dev.up(None if kw.get(n) is None else np.broadcast_to(np.asarray(kw[n]), rows), I32 if n == "top_k" else F32)
               for n in ("temp", "top_k", "top_p", "min_p")}
        if pad:
            wide = np.full((rows, V + pad), 1e4, x.dtype)
            wide[:, :V] = x
            x = wide
        ids, prob = dev.up(np.full(rows, -7, I32)), dev.up(np.full(rows, -7, F32))
        ctx.sample(dev.up(x), rows, V, dev.up(u, F32), ids, f16=x.dtype == F16, x_stride=0 if one_row else V + pad, prob=prob, **arr)
        return dev.get(ids, rows, I32), dev.get(prob, rows, F32)


def check_sample(ctx, x, u, **kw):
    """ids equal; probabilities rounded to fp32. Sums are counted in 2^-S of the largest weight (S >= 62 - log2 V): a border
    between two tokens is off by 2^-(S + 1) per token at most, and where u is no farther than that from one the oracle's
    own sum does not decide either; no u of these tests is (asserted)."""
    rows, V = len(u), x.shape[-1]
    ids, prob = run_sample(ctx, x, u, **kw)
    per = {n: np.broadcast_to(np.asarray(kw[n]), rows) for n in ("temp", "top_k", "top_p", "min_p") if kw.get(n) is not None}
    for r in range(rows):
        row = x[0] if kw.get("one_row") else x[r]
        a = {n: (int if n == "top_k" else F32)(p[r]) for n, p in per.items()}
        want, p, near = ref.sample(row, F32(u[r]), **a)
        if ids[r] != want:
            assert near < V * 2.0 ** -45, (r, ids[r], want, near, a)
            raise AssertionError((r, "u on a border", near))
        if np.isnan(p):
            assert np.isnan(prob[r])
        else:
            assert abs(prob[r] - p) <= 2.0 ** -24 * p + 2.0 ** -40, (r, prob[r], p)
    return ids, prob


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 2025, 4097, 8192, 16385, 50257, 128001])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_sample(ctx, V, dtype):
    print(f"sample {V}", flush=True)
    rng = np.random.default_rng(V)
    rows = 12 if V < 20000 else 6
    x = (rng.standard_normal((rows, V)) * 3).astype(dtype)
    u = rng.random(rows).astype(F32)
    temp = (0.4 + rng.random(rows)).astype(F32)
    check_sample(ctx, x, u)
    check_sample(ctx, x, u, temp=temp)
    for k in (1, 2, 40, V // 2, V - 1, V, V + 5, 0, -3):
        check_sample(ctx, x, u, temp=temp, top_k=k)
    for p in (0.0, -1.0, 0.01, 0.5, 0.9, 0.999999, 1.0, 2.0):
        check_sample(ctx, x, u, temp=temp, top_p=p)
    for p in (0.0, -1.0, 1e-6, 0.05, 0.9, 1.0, 3.0):
        check_sample(ctx, x, u, temp=temp, min_p=p)
    mixed = dict(top_k=rng.integers(0, V + 1, rows), top_p=rng.random(rows).astype(F32) * 1.2, min_p=(rng.random(rows) * 0.3).astype(F32))
    check_sample(ctx, x, u, temp=np.where(np.arange(rows) % 5 == 3, 0, temp), **mixed)


@pytest.mark.parametrize("V", [300, 2025, 20001])
@pytest.mark.parametrize("spread", [0.0, 0.02, 0.5, 12.0])
def test_sample_flat_and_peaked_rows(ctx, V, spread):
    """all equal, many equal (fp16 in a narrow range), nearly all the weight in one token"""
    rng = np.random.default_rng(V)
    for dtype in (F32, F16):
        x = (rng.standard_normal((6, V)) * spread + 3).astype(dtype)
        u = rng.random(6).astype(F32)
        for kw in ({}, {"top_k": V // 3}, {"top_p": 0.37}, {"top_k": V // 2, "top_p": 0.61}, {"min_p": 0.5}, {"top_p": 0.9999, "min_p": 0.01},
                   {"temp": 1e-3, "top_p": 0.5}, {"temp": 1e6, "top_k": 7}, {"top_k": 5000, "top_p": 0.3}):
            check_sample(ctx, x, u, **kw)


def test_sample_every_token_of_a_row(ctx):
    """one row, many draws: each kept token comes where its running sum says, the others never"""
    rng = np.random.default_rng(2)
    n = 4000
    x = (rng.standard_normal((1, 200)) * 1.5).astype(F32)
    u = ((np.arange(n) + 0.5) / n).astype(F32)
    for kw in ({}, {"top_k": 30}, {"top_p": 0.8}, {"min_p": 0.1}, {"top_k": 50, "top_p": 0.9, "min_p": 0.02, "temp": 1.3}):
        ids, _ = check_sample(ctx, x, u, one_row=True, **kw)
        w = ref.kept(x[0], **{k: (F32(v) if k != "top_k" else v) for k, v in kw.items()})
        assert (np.diff(ids) >= 0).all() and set(ids) <= set(np.nonzero(w)[0])
        big = np.nonzero(w / w.sum() > 2 / n)[0]
        assert set(big) <= set(ids)


def test_sample_exact_borders(ctx):
    """weights that are powers of two: u on a border takes the next token; top-p reached exactly ends there; ties by id"""
    x = np.log(np.array([[1, 1, 2, 4, 8, 0.5, 0.5, 1]])).astype(F32) * 0
    x[:] = np.array([0, 0, 1, 2, 3, -1, -1, 0])
    T = F32(1.4426950408889634)                        # exp(l / T) = 2^l to a rounding of T's
    u = np.array([0, 0.25, 0.5, 0.75, 0.999, 1.0, 2.0, -1.0, np.nan], F32)
    ids, _ = run_sample(ctx, np.repeat(x * 0, 9, 0), u)
    assert ids.tolist() == [0, 2, 4, 6, 7, 7, 7, 0, 0]
    ids, _ = run_sample(ctx, np.repeat(x * 0, 9, 0), u, top_p=0.5)
    assert ids.tolist() == [0, 1, 2, 3, 3, 3, 3, 0, 0]
    ids, _ = run_sample(ctx, np.repeat(x * 0, 9, 0), u, top_k=2)
    assert ids.tolist() == [0, 0, 1, 1, 1, 1, 1, 0, 0]
    ids, prob = run_sample(ctx, np.repeat(x, 2, 0), np.array([0.3, 0.99], F32), top_k=2, temp=T)
    assert ids.tolist() == [3, 4] and np.allclose(prob, [1 / 3, 2 / 3], atol=1e-6)
    zero = np.array([[0.0, -0.0, 0.0, -0.0]], F32)     # equal
    assert run_sample(ctx, np.repeat(zero, 2, 0), np.array([0.2, 0.7], F32), top_k=2)[0].tolist() == [0, 1]


@pytest.mark.parametrize("V", [9, 3000, 40000])
def test_sample_special_values(ctx, V):
    rng = np.random.default_rng(3)
    low = np.finfo(F32).min
    x = rng.standard_normal((9, V)).astype(F32)
    x[0] = -np.inf
    x[1, 5] = np.nan
    x[2, 3], x[2, 7] = np.inf, np.inf
    x[3], x[3, 4] = -np.inf, -1e30
    x[4], x[4, 2:6] = low, low
    x[5, ::2] = -np.inf
    x[6, :8] = 3e38
    x[7], x[7, 8] = -np.inf, 1.0
    x[8, V // 2] = np.inf
    u = np.array([.5, .5, .7, .5, .3, .6, .99, .5, .1], F32)
    for kw in ({}, {"top_k": 4}, {"top_p": 0.7}, {"min_p": 0.2}, {"temp": np.inf}, {"temp": 0.0}, {"temp": -1.0}, {"temp": np.nan}, {"temp": 1e-30}, {"top_p": np.nan, "min_p": np.nan},
               {"top_k": 3, "top_p": 0.9, "min_p": 0.1, "temp": 2.0}):
        check_sample(ctx, x, u, **kw)
    ids, prob = run_sample(ctx, x, u)
    assert ids[:2].tolist() == [-1, -1] and prob[0] == 0 and np.isnan(prob[1]) and ids[2] == 7 and ids[8] == V // 2


# min-p, largest logit, temperature, and two logits next to each other's weight: in 64 bits the lower one weighs min-p and the
# higher one 2^-53 less (computed weights are within 2^-51 of theirs, and do not all fall with the logits)
MIN_P_BORDERS = [("0x1.a3f7ccp-1", "0x1.7816bep+0", "0x1.da825ep+2", "0x1.87e6cp-34", "0x1.87e78p-34"),
                 ("0x1.8689d2p-1", "0x1.57fd6ap+0", "0x1.3d91fp+2", "0x1.ac008p-34", "0x1.ac01p-34"),
                 ("0x1.7797fcp-1", "0x1.05c666p+0", "0x1.a677b2p+1", "-0x1.8ba8p-35", "-0x1.8ba78p-35")]


@pytest.mark.parametrize("V", [300, 5000, 8193, 40000])
@pytest.mark.parametrize("border", MIN_P_BORDERS)
def test_sample_weights_that_are_min_p(ctx, V, border):
    """tokens whose weight is min-p to the last bit are all kept or all left out, and one of what is kept is drawn"""
    print(f"sample min-p {V} {border[0]}", flush=True)
    p, m, T, low, high = (F32(float.fromhex(t)) for t in border)
    u = np.array([0, 0.1234, 0.37, 0.5617, 0.777, 0.9123, 0.98765, 0.99999], F32)
    for kind in range(3):
        x = np.full((1, V), (low, high, low)[kind], F32)
        if kind == 2:
            x[0, ::2] = high
        x[0, 5] = m
        ids, prob = run_sample(ctx, x, u, one_row=True, temp=T, min_p=p)
        w = np.exp((x[0].astype(F64) - F64(m)) / F64(T))
        sets = [np.arange(V) == 5, np.ones(V, bool), x[0] != high, x[0] != low]         # of which one is kept
        fits = []
        for keep in sets:
            run = np.cumsum(w * keep)
            at = np.searchsorted(run, u.astype(F64) * run[-1], side="right")
            fits.append(np.array_equal(ids, at) and np.allclose(prob, w[at] / run[-1], rtol=1e-6))
        assert any(fits), (kind, ids, prob)


def test_sample_rows_apart_and_without_options(ctx):
    rng = np.random.default_rng(4)
    for V, pad in ((1001, 23), (30000, 1)):
        for dtype in (F32, F16):
            x, u = rng.standard_normal((5, V)).astype(dtype), rng.random(5).astype(F32)
            ids, prob = run_sample(ctx, x, u, top_k=9)
            got = run_sample(ctx, x, u, top_k=9, pad=pad)
            assert np.array_equal(got[0], ids) and np.array_equal(got[1], prob)
            with Dev(ctx) as dev:
                out = dev.up(np.zeros(5, I32))
                ema.lib().mgh_sample(ctx.h, dev.up(x).p, int(dtype == F16), V, 5, V, None, dev.up(u).p, out.p, None)
                assert np.array_equal(dev.get(out, 5, I32), run_sample(ctx, x, u)[0])


@pytest.mark.parametrize("rows,V", [(400, 128001), (170, 300001)])
def test_sample_rows_past_one_workspace(ctx, rows, V):
    """more rows than the workspace holds at a time (371 and 160): each as by itself"""
    print(f"sample batches {rows} {V}", flush=True)
    rng = np.random.default_rng(V)
    x = rng.standard_normal((rows, V), dtype=F32) * F32(2)
    u = rng.random(rows).astype(F32)
    k, p, T = rng.integers(1, 2000, rows).astype(I32), (rng.random(rows) * 0.9 + 0.1).astype(F32), (0.5 + rng.random(rows)).astype(F32)
    with Dev(ctx) as dev:
        dx, du, dk, dp, dt = dev.up(x), dev.up(u), dev.up(k), dev.up(p), dev.up(T)
        ids, prob = dev.up(np.full(rows, -7, I32)), dev.up(np.full(rows, -7, F32))
        ctx.sample(dx, rows, V, du, ids, temp=dt, top_k=dk, top_p=dp, prob=prob)
        got, gp = dev.get(ids, rows, I32), dev.get(prob, rows, F32)
    for r in sorted({*range(0, rows, 23), 159, 160, rows - 1} | {r for r in (370, 371) if r < rows}):
        one = run_sample(ctx, x[r:r + 1], u[r:r + 1], top_k=k[r], top_p=p[r], temp=T[r])
        assert got[r] == one[0][0] and gp[r] == one[1][0], r
    check_sample(ctx, x[-1:], u[-1:], top_k=k[-1:], top_p=p[-1:], temp=T[-1:])


def test_sample_many_rows(ctx):
    """what a row gives does not depend on the others, nor on the call"""
    rng = np.random.default_rng(5)
    for rows, V in ((1500, 700), (300, 5000), (70, 33000)):
        x = (rng.standard_normal((rows, V)) * 2).astype(F32)
        u = rng.random(rows).astype(F32)
        kw = dict(top_p=np.full(rows, 0.8, F32), temp=(0.5 + rng.random(rows)).astype(F32))
        ids, prob = run_sample(ctx, x, u, **kw)
        for _ in range(2):
            again = run_sample(ctx, x, u, **kw)
            assert np.array_equal(again[0], ids) and np.array_equal(again[1], prob)
        for r in range(0, rows, rows // 7):
            one = run_sample(ctx, x[r:r + 1], u[r:r + 1], top_p=0.8, temp=kw["temp"][r:r + 1])
            assert one[0][0] == ids[r] and one[1][0] == prob[r]
            assert ref.sample(x[r], u[r], top_p=F32(0.8), temp=kw["temp"][r])[0] == ids[r]


# ---- together -----------------------------------------------------------------------------


def test_generating_from_a_shared_prompt(ctx):
    """a prompt that three sequences go on from: its keys rotated into shared pages once, then steps of rotation, appending,
    attention over shared and own blocks, head, penalties and draws, captured once and replayed, against the same steps in 64
    bits from the tokens that were drawn"""
    rng = np.random.default_rng(21)
    B, P, T, V, H, Hkv, D = 3, 64, 40, 300, 4, 2, 32
    E, w = H * D, (H + 2 * Hkv) * D
    pairs, f = [16], freqs_of([16])
    table_q = (rng.standard_normal((V, w)) * 0.8).astype(F32)
    head = rng.standard_normal((V, E)).astype(F32)
    prompt = rng.integers(0, V, P).astype(I32)
    with Dev(ctx) as dev:
        c = Cache(dev, B, Hkv, D, 4, rng)
        table = c.table.copy()
        table[:, :2] = table[0, :2]
        c.set_table(table)
        rot = ema.Rope(pairs, f)
        x = table_q[prompt][None].reshape(1, P, H + 2 * Hkv, D)
        # the prompt once, as sequence 0's; the others start on its pages
        first = ema.Kv8(c.k, c.v, c.scales, c.kt, c.vt, c.dtable, c.nb, c.pages, Hkv, D, 1)
        dx, st = dev.up(x), (1, w, D, P * w)
        qo = dev.up(np.zeros((1, P, H, D), F16))
        ctx.kv8_append_rope(first, rot, dx.ptr + 4 * E, dx.ptr + 4 * (E + Hkv * D), st, P, dev.up([0], I32), in16=False, q=dx, q_strides=st, H=H,
                            q_out=qo, qo_strides=(1, E, D, P * E))
        lens = dev.up(np.full(B, P, I32))
        rows, att, qr = dev.up(np.zeros((B, w), F32)), dev.up(np.zeros((B, E), F32)), dev.up(np.zeros((B, E), F16))
        lg, y = dev.up(np.zeros((B, V), F32)), dev.up(np.zeros((B, V), F32))
        dt, dh, ids = dev.up(table_q), dev.up(head), dev.up(np.full(B, prompt[-1], I32))
        u, prob = dev.up(np.zeros(B, F32)), dev.up(np.zeros(B, F32))
        opts = {n: dev.up(np.full(B, a, t)) for n, a, t in (("temp", 4.0, F32), ("top_k", 50, I32), ("top_p", 0.9, F32))}
        hist, hlen, pres = dev.up(np.zeros((B, T), I32)), dev.up(np.zeros(B, I32)), dev.up(np.full(B, 0.7, F32))
        shared = dev.up([2], I32)
        st1, ost1 = (1, w, D, w), (1, E, D, E)

        def step():
            ctx.get_rows(dt, w, V, ids, B, rows)
            ctx.kv8_append_rope(c.h, rot, rows.ptr + 4 * E, rows.ptr + 4 * (E + Hkv * D), st1, 1, lens, in16=False, q=rows, q_strides=st1, H=H,
                                q_out=qr, qo_strides=ost1)
            ctx.kv8_attn_shared(c.h, qr, ost1, 1, lens, None, B, shared, 2, H, D ** -0.5, o=att, o_strides=ost1)
            ctx.gemm_f32(dh, V, E, att, B, None, 0, None, lg)
            ctx.logits_process(lg, B, V, y, hist=hist, max_hist=T, hist_len=hlen, pres=pres)
            ctx.sample(y, B, V, u, ids, prob=prob, **opts)
            ctx.kv8_advance(lens, None, B, 1)

        seqs, past = [list(prompt) for _ in range(B)], [[] for _ in range(B)]
        tok, graph = np.full(B, prompt[-1], I32), None
        draws = rng.random((T, B)).astype(F32)
        for t in range(T):
            ctx.write(u, draws[t])
            ctx.write(hist, np.array([p + [0] * (T - len(p)) for p in past], I32))
            ctx.write(hlen, np.array([len(p) for p in past], I32))
            if t == 1:
                ctx.graph_begin()
                step()
                graph = ctx.graph_end()
            graph.launch() if graph else step()
            got, new = dev.get(y, (B, V), F32), dev.get(ids, B, I32)
            assert dev.get(lens, B, I32).tolist() == [P + t + 1] * B
            for b in range(B):
                seqs[b].append(int(tok[b]))
                past[b].append(int(tok[b]))
                rows64 = table_q[seqs[b]].reshape(1, -1, H + 2 * Hkv, D)
                n = rows64.shape[1]
                at = np.arange(n)[None, None]
                kk = gen.cache_values(ref.rope(rows64[:, :, H:H + Hkv], at, pairs, f, 0)[0].astype(F16))
                vv = gen.cache_values(rows64[0, :, H + Hkv:].astype(F16))
                qq = ref.rope(rows64[:, :, :H], at, pairs, f, 0)[0, -1].astype(F16).astype(F64)
                a = np.stack([gen.attention_row(qq[h], kk[:, h // 2], vv[:, h // 2], D ** -0.5, 0.0, None, n - 1, np.ones(n, bool)) for h in range(H)])
                want = head.astype(F64) @ a.ravel()
                one, _ = gen.logits(want[None], hist=np.array([past[b][:-1] + [0]], I32), hist_len=[len(past[b]) - 1], pres=[0.7])
                # a rotated value may round to the neighbouring fp16 number (2^-10 of it) and its code to the next (1 / 127 of its
                # block's largest): far less than that on average; logits are sums of E such outputs
                assert np.abs(got[b] - one[0]).max() <= 0.02 * np.abs(one[0]).max(), np.abs(got[b] - one[0]).max()
                # the draw from the logits that the device had
                assert new[b] == ref.sample(got[b], draws[t, b], temp=F32(4), top_k=50, top_p=F32(0.9))[0]
            tok = new
        assert len({tuple(p) for p in past}) == B                # three different continuations
        graph.destroy()


def test_capture_and_replay_of_each(ctx):
    """each operator captured, replayed with eager work between, beside a second context's stream"""
    rng = np.random.default_rng(31)
    group, shared, own, new, H, Hkv, D = 6, [9], [5, 0, 33, 7, 60, 1], [1] * 6, 8, 2, 64
    with Dev(ctx) as dev, ema.Context(0) as other:
        c, q, k, v, lens, have, _ = shared_case(dev, rng, group, shared, own, new, H, Hkv, D)
        V = 40001
        x = (rng.standard_normal((6, V)) * 2).astype(F32)
        dx, du, dk, dp = dev.up(x), dev.up(rng.random(6), F32), dev.up(np.full(6, 300, I32)), dev.up(np.full(6, 0.8, F32))
        dq, dl, ds = dev.up(q), dev.up(lens, I32), dev.up(shared, I32)
        st = (1, H * D, D, H * D)
        rot = ema.Rope([16, 16], freqs_of([16, 16]))
        outs = [[dev.up(np.zeros(q.shape, F16)), dev.up(np.zeros(q.shape, F32)), dev.up(np.zeros(6, I32)), dev.up(np.zeros(6, F32))] for _ in range(2)]

        def work(cx, o):
            cx.rope(rot, dq, st, D, 1, H, 6, y16=o[0], y_strides=st, first=dl)
            cx.kv8_attn_shared(c.h, o[0], st, 1, dl, None, group, ds, 9, H, 0.125, o=o[1], o_strides=st)
            cx.sample(dx, 6, V, du, o[2], top_k=dk, top_p=dp, prob=o[3])

        def values(o):
            return [dev.get(b, n, t) for b, n, t in zip(o, (q.size, q.size, 6, 6), (F16, F32, I32, F32))]

        work(ctx, outs[0])
        want = values(outs[0])
        work(other, outs[1])
        other.sync()
        ctx.graph_begin()
        work(ctx, outs[0])
        g = ctx.graph_end()
        for rep in range(4):
            for b, n, t in zip(outs[0], want, (F16, F32, I32, F32)):
                ctx.write(b, np.zeros(n.shape, t))
            g.launch()
            work(other, outs[1])
            if rep % 2:
                work(ctx, outs[0])
            for a, b in zip(values(outs[0]), want):
                assert np.array_equal(a, b)
            other.sync()
            for a, b in zip(values(outs[1]), want):
                assert np.array_equal(a, b)
        g.destroy()
