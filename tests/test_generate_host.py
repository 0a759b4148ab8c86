"""The host side of the operators of token-by-token generation without a GPU: what each call refuses, and
that a refused or empty call launches nothing, on the recording HIP runtime of tests/test_dispatch.py."""
import numpy as np
import pytest

import edge_maskgit_amd as ema
from tests import gen_oracle as ref
from tests.test_dispatch import fake_hip, run  # noqa: F401 (the fixture builds the runtime)

BODY = """
def refused(f, *a, **kw):
    what = kw.pop("what")
    try:
        f(*a, **kw)
    except ema.MghError as e:
        assert what in str(e), (what, str(e))
        assert not kernels()
        return
    raise SystemExit("accepted: %s" % what)

def nothing(f, *a, **kw):
    f(*a, **kw)
    assert not kernels()
"""


def test_masked_attention_refusals():
    run(BODY + """
st = (1, 64, 16, 64 * 9)
def call(q=W, k=X, v=B, q_st=st, kv_st=st, D=16, Sq=9, Sk=9, H=4, Hkv=4, Bn=2, scale=0.25, o16=Y, **kw):
    c.attn_masked(q, k, v, q_st, kv_st, D, Sq, Sk, H, Hkv, Bn, scale, o16=o16, **kw)
call()
assert kernels()
nan = float("nan")
for kw, what in (({"D": 24}, "D must"), ({"D": 144}, "D must"), ({"D": 0}, "D must"), ({"H": 3, "Hkv": 2}, "H % Hkv"),
                 ({"Hkv": 0}, "H % Hkv"), ({"H": -4}, "H % Hkv"), ({"scale": nan}, "scale"), ({"scale": float("inf")}, "scale"),
                 ({"cap": -1.0}, "cap"), ({"cap": nan}, "cap"), ({"cap": float("inf")}, "cap"), ({"cap": 1e-45}, "fp32"), ({"cap": 3e38}, "fp32"), ({"scale": 3e38}, "fp32"), ({"o16": None}, "exactly one"),
                 ({"o": G}, "exactly one"), ({"Sq": -1}, "negative"), ({"Sk": -1}, "negative"), ({"Bn": -1}, "negative"),
                 ({"prefix": R}, "needs causal"), ({"docs": R, "doc_stride": 8}, "doc_stride"), ({"docs": R, "doc_stride": -9}, "doc_stride"),
                 ({"q": None}, "null"), ({"k": None}, "null"), ({"v": None}, "null"), ({"q": W + 1}, "aligned"), ({"o16": Y + 1}, "aligned"),
                 ({"v": B + 2, "in16": False}, "aligned"), ({"slopes": R + 2}, "aligned"), ({"docs": R + 1, "doc_stride": 9}, "aligned"),
                 ({"Sk": 2 ** 24 + 1}, "at most"), ({"Bn": 65536}, "at most"), ({"H": 70000, "Hkv": 70000}, "at most")):
    refused(call, what=what, **kw)
L = ema.lib()
assert L.mgh_attn_masked(c.h, W, X, B, 2, (ctypes.c_int64 * 4)(*st), (ctypes.c_int64 * 4)(*st), 16, 9, 9, 4, 4, 2, 0.25, None, None, Y, None) == -1
assert L.mgh_attn_masked(c.h, W, X, B, 1, None, None, 16, 9, 9, 4, 4, 2, 0.25, None, None, Y, None) == -1
assert L.mgh_attn_masked(None, W, X, B, 1, None, None, 16, 9, 9, 4, 4, 2, 0.25, None, None, Y, None) == -1
nothing(call, Sq=0)
nothing(call, Bn=0)
call(Sk=0, k=None, v=None)                       # rows of zeros
assert kernels()
""")


def test_cache_refusals():
    run(BODY + """
def kv(k=W, v=X, scales=B, kt=R, vt=Y, table=G, nb=4, pages=9, Hkv=2, D=32, Bn=3, **kw):
    return ema.Kv8(k, v, scales, kt, vt, table, nb, pages, Hkv, D, Bn, **kw)
Q, O, N = (0x100000 * i for i in (17, 18, 19))
st = (1, 64, 32, 64 * 5)
calls = {
    "append": lambda h, S=5, lens=N, k=Q, v=Q, **kw: c.kv8_append(h, k, v, st, S, lens, **kw),
    "attn": lambda h, S=5, lens=N, q=Q, H=2, scale=0.1, o16=O, **kw: c.kv8_attn(h, q, st, S, lens, None, H, scale, o16=o16, **kw),
    "read": lambda h, S=5, lens=N, k=Q, v=Q, **kw: c.kv8_read(h, None, S, lens, k=k, v=v, **kw)}
for name, f in calls.items():
    f(kv())
    assert kernels(), name
    nothing(f, kv(), S=0)
    nothing(f, kv(Bn=0))
    for kw, what in (({"Hkv": 0}, "Hkv, D > 0"), ({"D": 20}, "D must"), ({"D": 160}, "D must"), ({"D": -16}, "Hkv, D > 0"), ({"Bn": -1}, "negative"),
                     ({"pages": -1}, "negative"), ({"nb": -1}, "negative"), ({"table_stride": 3}, "table_stride"), ({"Hkv": 70000}, "65535"),
                     ({"Bn": 70000}, "65535"), ({"nb": 2 ** 24 + 1}, "2^24"), ({"pages": 2 ** 31}, "pages"), ({"k": None}, "null"), ({"v": None}, "null"),
                     ({"scales": None}, "null"), ({"kt": None}, "null"), ({"vt": None}, "null"), ({"table": None}, "null"), ({"k": W + 8}, "aligned"),
                     ({"vt": Y + 2}, "aligned"), ({"scales": B + 4}, "aligned"), ({"table": G + 2}, "aligned")):
        refused(f, kv(**kw), what=what)
    refused(f, kv(), S=-1, what="negative")
    refused(f, kv(), S=2 ** 28 + 1, what="2^28")
    refused(f, kv(), lens=None, what="null")
    refused(f, kv(), lens=N + 2, what="aligned")
refused(calls["append"], kv(), k=None, what="null")
refused(calls["append"], kv(), v=Q + 2, in16=False, what="aligned")
refused(calls["append"], kv(), k=Q + 1, what="aligned")
for kw, what in (({"H": 3}, "H % Hkv"), ({"H": 0}, "H % Hkv"), ({"scale": float("nan")}, "scale"), ({"cap": -2.0}, "cap"), ({"o": W}, "exactly one"),
                 ({"o16": None}, "exactly one"), ({"q": None}, "null"), ({"q": Q + 1}, "aligned"), ({"slopes": N + 1}, "aligned"), ({"S": 2 ** 24 + 1}, "2^24")):
    refused(calls["attn"], kv(), what=what, **kw)
refused(calls["read"], kv(), v=None, what="either")
refused(calls["read"], kv(), k16=O, v16=O, what="either")
refused(calls["read"], kv(), k=Q + 2, what="aligned")
refused(c.kv8_advance, None, None, 3, 1, what="null")
refused(c.kv8_advance, N, None, -1, 1, what="negative")
refused(c.kv8_advance, N, None, 3, -1, what="negative")
nothing(c.kv8_advance, N, None, 0, 1)
c.kv8_advance(N, None, 3, 1)
assert kernels() == ["k_kv8_advance"]
assert ema.lib().mgh_kv8_append(c.h, None, Q, Q, 1, (ctypes.c_int64 * 4)(*st), 1, N, None) == -1
assert ema.lib().mgh_kv8_attn(c.h, ctypes.byref(kv()), Q, 1, None, 1, N, None, 2, 0.1, 0.0, None, None, O, None) == -1
assert ema.kv8_code_bytes(9, 2, 32) == 9 * 2 * 32 * 32 and ema.kv8_scale_bytes(9, 2) == 9 * 2 * 8
assert ema.kv8_tail_bytes(3, 2, 32) == 3 * 2 * 32 * 64 * 2 and ema.kv8_code_bytes(-1, 2, 32) == ema.kv8_tail_bytes(3, 0, 32) == 0
""")


def test_logits_refusals():
    run(BODY + """
def call(x=W, rows=3, V=1000, y=Y, **kw):
    c.logits_process(x, rows, V, y, **kw)
call()
assert kernels()
call(y=W)
call(rows=1, x_stride=0, y_stride=0)
kernels()
for kw, what in (({"x": None}, "null"), ({"y": None}, "null"), ({"rows": -1}, "negative"), ({"V": -1}, "negative"), ({"V": 2 ** 30 + 1}, "too large"),
                 ({"rows": 2 ** 30}, "too large"), ({"x_stride": 999}, "apart"), ({"y_stride": 10}, "apart"), ({"y": W, "x_stride": 1001}, "equal strides"),
                 ({"hist": R, "max_hist": -1}, "negative"), ({"hist": R, "max_hist": 9, "hist_stride": 8}, "hist_stride"),
                 ({"bias": R, "bias_stride": 999}, "bias_stride"), ({"bias": R, "bias_stride": -1}, "negative"),
                 ({"allowed": R, "allowed_stride": 31}, "allowed_stride"), ({"x": W + 2}, "aligned"), ({"y": Y + 1, "f16": True}, "aligned"),
                 ({"rep": R + 1}, "aligned"), ({"hist_len": R + 2}, "aligned")):
    refused(call, what=what, **kw)
nothing(call, rows=0)
nothing(call, V=0)
""")


def test_oracle_quantization_is_the_exact_rounding():
    """the oracle's codes against whole-number arithmetic: |x| / d in units of fp16's and fp32's last places"""
    from fractions import Fraction
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(400) * 3).astype(np.float16)
    codes, d = ref.quantize(x)
    assert d == np.float32(np.abs(x).max()) / np.float32(127)
    for a, c in zip(x.tolist(), codes.tolist()):
        t = Fraction(abs(a)) / Fraction(float(d))
        want = int(t + Fraction(1, 2))                   # halves away from zero
        assert c == (want if a >= 0 else -want)
    assert np.abs(codes).max() == 127


def test_entry_points_take_no_context():
    L = ema.lib()
    assert L.mgh_kv8_advance(None, None, None, 1, 1) == -1
    assert L.mgh_logits_process(None, None, 0, 1, 1, 1, None, None, 1) == -1
    assert L.mgh_kv8_read(None, None, None, 1, None, None, None, None, None) == -1


@pytest.mark.parametrize("cap", [0.0, 2.0])
def test_oracle_matches_a_plain_softmax(cap):
    """the row oracle against the formula written out, with every key seen"""
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal(8), rng.standard_normal((20, 8)), rng.standard_normal((20, 8))
    s = k @ q * 0.3
    s = cap * np.tanh(s / cap) if cap else s
    s = s - 0.1 * np.abs(19 - np.arange(20))
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(ref.attention_row(q, k, v, 0.3, cap, 0.1, 19, np.ones(20, bool)), w @ v, atol=1e-12)


def test_which_kernels_masked_attention_takes():
    """tiles per wave, parts of the keys, packing and joining, as the rules say"""
    run(BODY + """
def call(Sq, Sk, H, Hkv, D, Bn=1, in16=True, out16=True, q=W, st=None, **kw):
    q_st = st or (1, H * D, D, Sq * H * D)
    launches()
    c.attn_masked(q, X, B, q_st, (1, Hkv * D, D, Sk * Hkv * D), D, Sq, Sk, H, Hkv, Bn, D ** -0.5, in16=in16,
                  **{"o16" if out16 else "o": Y}, **kw)
    return launches()

def tile(l):
    m = re.search(r"k_attn_maskedILi(\\d)ELi(\\d)ELb(\\d)ELi(\\d)E", l[1])
    return tuple(map(int, m.groups())), l[2][0]

def one(*a, **kw):
    l = call(*a, **kw)
    assert [k for k, _, _ in l] == ["k_attn_masked"], l
    return tile(l[0])

# many rows: two 16-row tiles per wave for wide heads, and for narrow ones whose rows all see the same keys
assert one(4097, 4097, 32, 32, 128) == ((8, 2, 0, 0), 33 * 32)
assert one(4097, 4097, 32, 32, 128, causal=True) == ((8, 2, 0, 0), 33 * 32)
assert one(4097, 4097, 32, 32, 64) == ((4, 2, 0, 0), 33 * 32)
assert one(4097, 4097, 32, 32, 64, causal=True) == ((4, 1, 0, 0), 65 * 32)
assert one(4097, 4097, 32, 32, 64, docs=G, doc_stride=0) == ((4, 1, 0, 0), 65 * 32)
assert one(4097, 4097, 32, 32, 64, cap=30.0) == ((4, 1, 0, 2), 65 * 32)
# the heads of a group are rows of one tile
assert one(4096, 4096, 32, 8, 128) == ((8, 2, 0, 0), 128 * 8)
# scores: scaled, sloped or of any scale, capped, both or with caps past 64
assert one(257, 257, 16, 16, 48) == ((3, 1, 0, 0), 5 * 16)
assert one(257, 257, 16, 16, 48, slopes=R) == ((3, 1, 0, 1), 5 * 16)
assert one(257, 257, 16, 16, 48, cap=30.0) == ((3, 1, 0, 2), 5 * 16)
assert one(257, 257, 16, 16, 48, cap=70.0) == ((3, 1, 0, 3), 5 * 16)
assert one(257, 257, 16, 16, 48, cap=30.0, slopes=R) == ((3, 1, 0, 3), 5 * 16)
assert one(257, 257, 16, 16, 48, out16=False) == ((3, 1, 1, 0), 5 * 16)
for D, dc in ((16, 2), (32, 2), (80, 6), (96, 6), (112, 8)):
    assert one(64, 64, 2, 2, D) == ((dc, 1, 0, 0), 2)
# few workgroups: the keys in parts of at least four chunks, joined
for sk, parts, join in ((448, 1, None), (511, 2, "ILi2E"), (512, 2, "ILi2E"), (1000, 4, "ILi4E"), (2048, 8, "ILi8E"), (8192, 32, "k_attn_joinE")):
    l = call(1, sk, 8, 2, 128)
    assert tile(l[0]) == ((8, 1, 0, 0), 2 * parts), (sk, l)
    assert len(l) == (1 if join is None else 2) and (join is None or join in l[1][1]), (sk, l)
assert [k for k, _, _ in call(1, 8000, 32, 8, 128, Bn=8)] == ["k_attn_masked", "k_attn_join_few"]
assert len(call(512, 12345, 32, 8, 128, Bn=2)) == 2
# rows that are not fp16, not 16-byte aligned or without unit stride are packed first
p = ["k_attn_pack", "k_attn_masked"]
assert [k for k, _, _ in call(64, 64, 2, 2, 64, in16=False, out16=False)] == p
assert [k for k, _, _ in call(64, 64, 2, 2, 64, q=W + 2)] == p
assert [k for k, _, _ in call(64, 64, 2, 2, 64, st=(1, 132, 64, 64 * 132))] == p
assert call(64, 64, 2, 2, 64, q=W + 2)[0][2][1] == 1 and call(64, 64, 2, 2, 64, in16=False)[0][2][1] == 3
assert one(64, 64, 2, 2, 64, st=(1, 136, 64, 64 * 136)) == ((4, 1, 0, 0), 2)
""")


def test_which_kernels_cache_attention_takes():
    run(BODY + """
def call(S, H, Hkv, D, Bn, nb, **kw):
    kv = ema.Kv8(W, X, B, R, Y, G, nb, 1 << 20, Hkv, D, Bn)
    launches()
    c.kv8_attn(kv, 0x1200000, (1, H * D, D, S * H * D), S, 0x1300000, None, H, D ** -0.5, o16=0x1400000, **kw)
    l = launches()
    m = re.search(r"k_kv8_attnILi(\\d)ELi(\\d)ELb(\\d)ELb(\\d)E", l[0][1])
    return tuple(map(int, m.groups())), l[0][2][0], [k for k, _, _ in l[1:]]

few, many = ["k_attn_join_few"], ["k_attn_join"]
assert call(1, 32, 8, 128, 1, 8) == ((4, 1, 0, 0), 8, [])                     # eight blocks: one part
assert call(1, 32, 8, 128, 1, 9) == ((4, 1, 0, 0), 16, few)
assert call(1, 32, 8, 128, 1, 64) == ((4, 1, 0, 0), 8 * 8, few)
assert call(1, 32, 8, 128, 1, 4096) == ((4, 1, 0, 0), 8 * 32, many)           # a workgroup per CU
assert call(1, 32, 8, 128, 1, 16384) == ((4, 1, 0, 0), 8 * 96, many)
assert call(1, 32, 8, 128, 1, 1 << 24) == ((4, 1, 0, 0), 2048, many)          # no more than eight per CU
assert call(1, 32, 8, 128, 64, 96) == ((4, 1, 0, 0), 512, [])                 # enough workgroups: parts of long sequences only
assert call(1, 32, 8, 128, 64, 97) == ((4, 1, 0, 0), 1024, few)
assert call(1, 32, 8, 128, 64, 1 << 20) == ((4, 1, 0, 0), 2048, few)
assert call(4, 32, 8, 128, 64, 8) == ((4, 1, 0, 0), 512, [])                  # 16 rows of a key head: one tile
assert call(5, 32, 8, 128, 64, 8) == ((4, 2, 0, 0), 512, [])
assert call(9, 32, 8, 128, 64, 8) == ((4, 2, 0, 0), 1024, [])
for D, dg in ((16, 1), (32, 1), (48, 2), (64, 2), (80, 3), (96, 3), (112, 4)):
    assert call(1, 8, 8, D, 64, 8) == ((dg, 1, 0, 0), 512, [])
assert call(1, 8, 8, 64, 64, 8, cap=3.0)[0] == call(1, 8, 8, 64, 64, 8, slopes=0x1500000)[0] == (2, 1, 0, 1)
""")
