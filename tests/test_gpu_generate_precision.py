"""How many bits the attentions keep: rows against 64 bits with tolerances from each row's own terms
(gen_oracle.row_tolerance), narrow enough that softmax weights of 11 bits with an fp32 output, or a cap computed with
an error of the cap's size, would not pass; both are planted here in the oracle, on the CPU."""
import numpy as np
import pytest

from tests import gen_oracle as ref
from tests.test_gpu_generate import Dev, cache_case, ctx, qkv, run_masked  # noqa: F401

F16, F32, F64 = np.float16, np.float32, np.float64
LOG2E = 1.4426950408889634

# B, Sq, Sk, H, Hkv, D
SHAPES = [(2, 7, 9, 4, 2, 16), (1, 12, 12, 2, 1, 48), (1, 70, 70, 4, 2, 32), (1, 3, 700, 6, 2, 64), (1, 130, 257, 2, 1, 128), (1, 2, 2500, 2, 2, 16)]
KINDS = {"plain": {}, "cap2": {"cap": 2.5}, "cap30": {"cap": 30.0}, "cap50": {"cap": 50.0}, "cap100": {"cap": 100.0},
         "slopes": {"slope": 0.25}, "cap20 and slopes": {"cap": 20.0, "slope": 0.03125}}


def rows_of(shape, rng):
    B, Sq, Sk, H, Hkv, D = shape
    q, k, v = qkv(rng, *shape)
    for b in range(B):
        for i in range(Sq):
            for h in range(H):
                yield (b, i, h), q[b, i, h].astype(F64), k[b, :, h // (H // Hkv)].astype(F64), v[b, :, h // (H // Hkv)].astype(F64), Sk - Sq + i


def fp16_weights(q, k, v, scale, cap, slope, p, seen):
    """attention_row with weights of 11 bits"""
    at = np.nonzero(seen)[0]
    s = (k[at] @ q) * scale
    s = cap * np.tanh(s / cap) if cap else s
    s = s if slope is None else s - slope * np.abs(p - at)
    w = np.exp(s - s.max())
    w = (w * 128).astype(F16).astype(F64)
    return w @ v[at] / w.sum()


@pytest.mark.parametrize("kind", list(KINDS))
def test_the_tolerance_sees_weights_of_11_bits(kind):
    kw = KINDS[kind]
    cap, slope = kw.get("cap", 0.0), kw.get("slope")
    for shape in SHAPES[:2]:
        over = 0
        for _, q, k, v, p in rows_of(shape, np.random.default_rng(sum(shape))):
            seen = np.arange(len(k)) <= p
            want = ref.attention_row(q, k, v, len(q) ** -0.5, cap, slope, p, seen)
            tol = ref.row_tolerance(q, k, v, len(q) ** -0.5, cap, slope, p, seen)
            over = max(over, (np.abs(fp16_weights(q, k, v, len(q) ** -0.5, cap, slope, p, seen) - want) / tol).max())
        assert over > 2, (shape, over)


def capped_pairs(cap):
    """rows of two keys, one feature: scores q and -q, capped, so that the output is tanh(cap tanh(q / cap))"""
    q = np.zeros((1, 400, 1, 16), F16)
    q[0, :, 0, 0] = np.linspace(-1.2, 1.2, 400)
    k = np.zeros((1, 2, 1, 16), F16)
    k[0, :, 0, 0] = 1, -1
    return q, k, k.copy()


@pytest.mark.parametrize("cap", [20.0, 30.0, 50.0, 64.0])
def test_the_tolerance_sees_a_coarse_cap(cap):
    """1 - 2 / (e + 1) in fp32, every operation rounded correctly"""
    q, k, v = capped_pairs(cap)
    s = q[0, :, 0, 0].astype(F64)
    e = np.exp2((s * F64(F32(2 * LOG2E / cap))).astype(F32)).astype(F32)
    y = cap * (1 - 2 * (1 / (e + F32(1))).astype(F64)).astype(F32).astype(F64)
    over = 0
    for i in range(400):
        row = q[0, i, 0].astype(F64), k[0, :, 0].astype(F64), v[0, :, 0].astype(F64), 1.0, cap
        over = max(over, abs(np.tanh(y[i]) - ref.attention_row(*row, None, 0, np.ones(2, bool))[0]) / ref.row_tolerance(*row)[0])
    assert over > 1, over


def near(got, want, tol, what):
    over = (np.abs(got.astype(F64) - want) / tol).max()
    assert over <= 1, (what, over)
    return over


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("out16", [False, True])
def test_masked_rows_keep_their_bits(ctx, shape, kind, out16):
    kw = KINDS[kind]
    cap, slope = kw.get("cap", 0.0), kw.get("slope")
    H, D = shape[3], shape[5]
    got = run_masked(ctx, *qkv(np.random.default_rng(sum(shape)), *shape), out16=out16, causal=True, cap=cap,
                     slopes=None if slope is None else np.full(H, slope, F32))
    worst = 0
    for (b, i, h), q, k, v, p in rows_of(shape, np.random.default_rng(sum(shape))):
        seen = np.arange(len(k)) <= p
        args = q, k, v, D ** -0.5, cap, slope, p, seen
        worst = max(worst, near(got[b, i, h], ref.attention_row(*args), ref.row_tolerance(*args, out16=out16), (b, i, h)))
    print(f"{shape} {kind} out16={out16}: {worst:.2f} of the tolerance", flush=True)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [20.0, 30.0, 50.0, 64.0, 100.0])
def test_caps_keep_their_bits(ctx, cap):
    q, k, v = capped_pairs(cap)
    got = run_masked(ctx, q, k, v, out16=False, cap=cap, scale=1.0)
    worst = 0
    for i in range(400):
        args = q[0, i, 0].astype(F64), k[0, :, 0].astype(F64), v[0, :, 0].astype(F64), 1.0, cap
        worst = max(worst, near(got[0, i, 0], ref.attention_row(*args, None, 0, np.ones(2, bool)), ref.row_tolerance(*args), i))
    print(f"cap {cap}: {worst:.2f} of the tolerance", flush=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lens,new,H,Hkv,D,spare", [([3, 0, 20], [2, 1, 1], 4, 2, 16, 0), ([200, 33, 63], [3, 1, 2], 4, 1, 48, 1), ([1000], [9], 4, 2, 128, 70)])
@pytest.mark.parametrize("out16", [False, True])
def test_cached_rows_keep_their_bits(ctx, lens, new, H, Hkv, D, spare, kind, out16):
    kw = KINDS[kind]
    cap, slope = kw.get("cap", 0.0), kw.get("slope")
    rng = np.random.default_rng(sum(lens) + D)
    worst = 0
    with Dev(ctx) as dev:
        c, q, k, v, have = cache_case(dev, rng, lens, new, H, Hkv, D, spare=spare)
        got = c.attend(q, lens, new, out16=out16, cap=cap, slopes=None if slope is None else np.full(H, slope, F32))
        for b, n in enumerate(have):
            kk, vv = ref.cache_values(k[b, :n]), ref.cache_values(v[b, :n])
            for i in range(new[b]):
                for h in range(H):
                    g, p = h // (H // Hkv), lens[b] + i
                    args = q[b, i, h].astype(F64), kk[:, g], vv[:, g], D ** -0.5, cap, slope, p, np.arange(n) <= p
                    worst = max(worst, near(got[b, i, h], ref.attention_row(*args), ref.row_tolerance(*args, out16=out16), (b, i, h)))
    print(f"{lens} {kind} out16={out16}: {worst:.2f} of the tolerance", flush=True)
