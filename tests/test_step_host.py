"""The host side of rotary positions, rotated appending, attention over shared blocks and sampling without a GPU: what
each call refuses, that a refused or empty call launches nothing, and which kernels the others take, on the recording HIP
runtime of tests/test_dispatch.py."""
import os
import struct

import msgpack
import numpy as np
import pytest

import edge_maskgit_amd as ema
from tests import step_oracle as ref
from tests.test_dispatch import fake_hip, run  # noqa: F401 (the fixture builds the runtime)
from tests.test_generate_host import BODY

ROPE = BODY + """
F = [1.0] * 64
def rot(pairs=(8,), freqs=F, order=0, pos=None, **kw):
    return ema.Rope(pairs, freqs, order, pos, **kw)
"""


def test_rope_refusals():
    run(ROPE + """
st = (1, 64, 16, 64 * 9)
def call(r=None, x=W, x_st=st, D=16, S=9, H=4, Bn=2, y=Y, **kw):
    c.rope(rot() if r is None else r, x, x_st, D, S, H, Bn, y=y, **kw)
call()
assert kernels() == ["k_rope"]
call(y=None, y16=Y, in16=False)
call(x=W, y=W, in16=False)                          # in place
kernels()
big = rot()
big.axes = 5
none = rot()
none.axes = 0
for r, what in ((big, "1 to 4 axes"), (none, "1 to 4 axes"), (rot((9,)), "pairs"), (rot((-1,)), "pairs"), (rot((4, 5)), "more pairs"), (rot(order=3), "order"),
                (rot(order=-1), "order"), (rot(freqs=[float("nan")] * 8), "frequencies"), (rot(freqs=[float("inf")] * 8), "frequencies"),
                (rot(freqs=[1.0] * 7 + [16.5]), "frequencies"), (rot(pos=R + 2), "aligned")):
    refused(call, r, what=what)
for kw, what in (({"D": 15}, "even"), ({"D": 130}, "even"), ({"D": 0}, "even"), ({"S": -1}, "negative"), ({"H": -1}, "negative"), ({"Bn": -1}, "negative"),
                 ({"y": None}, "exactly one"), ({"y16": G}, "exactly one"), ({"x": None}, "null"), ({"x": W + 1}, "aligned"), ({"x": W + 2, "in16": False}, "aligned"),
                 ({"y": Y + 2}, "aligned"), ({"y": None, "y16": Y + 1}, "aligned"), ({"first": R + 1}, "aligned"), ({"new": R + 2}, "aligned"),
                 ({"y": W}, "in place"), ({"y": W, "in16": False, "y_strides": (1, 64, 16, 64 * 10)}, "in place"), ({"Bn": 65536}, "at most"), ({"H": 65536}, "at most"),
                 ({"S": 2 ** 28 + 1}, "at most"), ({"S": 2 ** 25 + 1}, "at most")):
    refused(call, what=what, **kw)
L = ema.lib()
four = (ctypes.c_int64 * 4)(*st)
r = rot()
assert L.mgh_rope(c.h, None, W, 1, four, 16, 9, 4, 2, None, None, Y, None, four) == -1
assert L.mgh_rope(c.h, ctypes.byref(r), W, 2, four, 16, 9, 4, 2, None, None, Y, None, four) == -1
assert L.mgh_rope(c.h, ctypes.byref(r), W, 1, None, 16, 9, 4, 2, None, None, Y, None, four) == -1
assert L.mgh_rope(None, ctypes.byref(r), W, 1, four, 16, 9, 4, 2, None, None, Y, None, four) == -1
r.h_freqs = None
refused(call, r, what="null frequencies")
for kw in ({"S": 0}, {"H": 0}, {"Bn": 0}):
    nothing(call, **kw)
call(rot((0,), []))                                 # nothing turns: a copy
assert kernels() == ["k_rope"]
try:
    ema.Rope((8,), [1.0] * 7)
    raise SystemExit("accepted")
except ema.MghError:
    pass
""")


def test_rotated_append_refusals():
    run(ROPE + """
def kv(k=W, v=X, scales=B, kt=R, vt=Y, table=G, nb=4, pages=9, Hkv=2, D=32, Bn=3, **kw):
    return ema.Kv8(k, v, scales, kt, vt, table, nb, pages, Hkv, D, Bn, **kw)
Q, O, N = (0x100000 * i for i in (17, 18, 19))
st = (1, 64, 32, 64 * 5)
qst = (1, 128, 32, 128 * 5)
def call(h=None, r=None, S=5, lens=N, k=Q, v=Q, **kw):
    c.kv8_append_rope(kv() if h is None else h, rot() if r is None else r, k, v, st, S, lens, **kw)
q = dict(q=O, q_strides=qst, H=4, q_out=O + 0x80000, qo_strides=qst)
call()
call(**q)
call(**dict(q, q_out=O))
assert kernels() == ["k_kv8_append_rope"] * 3
nothing(call, S=0)
nothing(call, kv(Bn=0))
for kw, what in (({"Hkv": 0}, "Hkv, D > 0"), ({"D": 20}, "D must"), ({"table_stride": 3}, "table_stride"), ({"kt": None}, "null"), ({"k": W + 8}, "aligned")):
    refused(call, kv(**kw), what=what)
refused(call, r=rot((17,)), what="pairs")
refused(call, r=rot(order=7), what="order")
for kw, what in (({"S": -1}, "negative"), ({"S": 2 ** 28 + 1}, "2^28"), ({"lens": None}, "null"), ({"lens": N + 2}, "aligned"), ({"k": None}, "null"), ({"v": None}, "null"),
                 ({"k": Q + 1}, "aligned"), (dict(q, q=O + 1), "aligned"), (dict(q, H=3), "H % Hkv"), (dict(q, H=0), "H % Hkv"), (dict(q, q_out=None), "null"),
                 (dict(q, q_strides=None), "null"), (dict(q, qo_strides=None), "null"), (dict(q, q_out=O + 1), "aligned"), (dict(q, q_out=O, in16=False), "in place"),
                 (dict(q, q_out=O, qo_strides=(1, 256, 32, 1280)), "in place"), (dict(q, H=70000), "65535")):
    refused(call, what=what, **kw)
assert ema.lib().mgh_kv8_append_rope(c.h, ctypes.byref(kv()), None, Q, Q, 1, (ctypes.c_int64 * 4)(*st), 1, N, None, None, None, 0, None, None) == -1
assert ema.lib().mgh_kv8_append_rope(None, ctypes.byref(kv()), ctypes.byref(rot()), Q, Q, 1, None, 1, N, None, None, None, 0, None, None) == -1
""")


def test_shared_attention_refusals():
    run(BODY + """
def kv(k=W, v=X, scales=B, kt=R, vt=Y, table=G, nb=4, pages=9, Hkv=2, D=32, Bn=3, **kw):
    return ema.Kv8(k, v, scales, kt, vt, table, nb, pages, Hkv, D, Bn, **kw)
Q, O, N, M = (0x100000 * i for i in (17, 18, 19, 20))
st = (1, 64, 32, 64 * 5)
def call(h=None, S=5, lens=N, q=Q, H=2, scale=0.1, o16=O, group=2, shared=M, most=3, **kw):
    c.kv8_attn_shared(kv() if h is None else h, q, st, S, lens, None, group, shared, most, H, scale, o16=o16, **kw)
call()
assert kernels()
nothing(call, S=0)
nothing(call, kv(Bn=0))
for kw, what in (({"Hkv": 0}, "Hkv, D > 0"), ({"D": 160}, "D must"), ({"table": None}, "null"), ({"vt": Y + 2}, "aligned")):
    refused(call, kv(**kw), what=what)
for kw, what in (({"H": 3}, "H % Hkv"), ({"scale": float("nan")}, "scale"), ({"cap": -2.0}, "cap"), ({"o": W}, "exactly one"), ({"o16": None}, "exactly one"),
                 ({"q": None}, "null"), ({"q": Q + 1}, "aligned"), ({"slopes": N + 1}, "aligned"), ({"S": 2 ** 24 + 1}, "2^24"), ({"group": 0}, "group"), ({"group": -3}, "group"),
                 ({"most": -1}, "max_shared"), ({"most": 5}, "max_shared"), ({"shared": None}, "null"), ({"shared": M + 2}, "aligned"), ({"lens": None}, "null"),
                 ({"S": 2 ** 23}, "2^24")):
    refused(call, what=what, **kw)
call(group=1000)                                    # one group
assert kernels()
big = kv(Hkv=2, Bn=65535, nb=4)
refused(call, big, S=512, what="2^24")
refused(call, kv(Hkv=256, Bn=65535, nb=4), S=1, H=256, what="too large")
assert ema.lib().mgh_kv8_attn_shared(None, ctypes.byref(kv()), Q, 1, None, 1, N, None, 1, M, 1, 2, 0.1, 0.0, None, None, O, None) == -1
""")


def test_shared_attention_refuses_what_its_join_cannot_launch():
    """the join takes 32 threads per row: rows up to 2^27 - 1, refused before anything is launched; fewer run"""
    run(BODY + """
Q, O, N, M = (0x100000 * i for i in (17, 18, 19, 20))
def call(Bn, S=1024, Hkv=16, D=16):
    c.kv8_attn_shared(ema.Kv8(W, X, B, R, Y, G, 4, 9, Hkv, D, Bn), Q, (1, D, D, D), S, N, None, 64, M, 3, Hkv, 0.1, o16=O)
launches()
refused(call, 8192, what="2^27")
refused(call, 16383, what="2^27")
assert launches() == []
call(8191)
g = {k: n for k, _, n in launches()}
assert [n[0] * 256 < 2 ** 32 for n in g.values()] == [True, True] and g["k_attn_join_few"][0] * 8 >= 8191 * 2 ** 14
""")


def test_sample_refusals():
    run(BODY + """
def call(x=W, rows=3, V=1000, u=X, ids=Y, **kw):
    c.sample(x, rows, V, u, ids, **kw)
call()
assert kernels()
call(x_stride=0)
call(rows=1, x_stride=7)
kernels()
for kw, what in (({"x": None}, "null"), ({"u": None}, "null"), ({"ids": None}, "null"), ({"rows": -1}, "negative"), ({"V": -1}, "negative"), ({"V": 0}, "without"),
                 ({"V": 2 ** 24 + 1}, "at most"), ({"rows": 2 ** 20 + 1}, "at most"), ({"x_stride": 999}, "x_stride"), ({"x_stride": -1000}, "x_stride"), ({"x": W + 2}, "aligned"),
                 ({"x": W + 1, "f16": True}, "aligned"), ({"u": X + 1}, "aligned"), ({"temp": R + 2}, "aligned"), ({"top_k": R + 2}, "aligned"),
                 ({"top_p": R + 1}, "aligned"), ({"min_p": R + 3}, "aligned"), ({"prob": R + 2}, "aligned"), ({"ids": Y + 2}, "aligned")):
    refused(call, what=what, **kw)
nothing(call, rows=0)
L = ema.lib()
assert L.mgh_sample(c.h, W, 2, 9, 1, 9, None, X, Y, None) == -1
assert L.mgh_sample(None, W, 0, 9, 1, 9, None, X, Y, None) == -1
""")


@pytest.mark.parametrize("order", [0, 1, 2])
def test_oracle_turns_every_feature_once(order):
    pairs = [3, 0, 2]
    seen = sorted(f for ab in ref.features(pairs, order) for f in ab)
    assert seen == list(range(10))
    x = np.random.default_rng(0).standard_normal((1, 4, 1, 12))
    pos = np.stack([np.arange(4)[None] * (a + 1) for a in range(3)])
    y = ref.rope(x, pos, pairs, [0.3, 0.2, 0.1, 1.0, 0.5], order)
    back = ref.rope(y, -pos, pairs, [0.3, 0.2, 0.1, 1.0, 0.5], order)
    assert np.allclose(back, x, atol=1e-12) and np.array_equal(y[..., 10:], x[..., 10:]) and np.array_equal(y[:, 0], x[:, 0])


def test_oracle_rotation_depends_on_the_distance():
    """products of a rotated query and key depend on the difference of their positions"""
    rng = np.random.default_rng(1)
    q, k = rng.standard_normal((2, 1, 1, 1, 8))
    f = [1.0, 0.1, 0.01, 0.001]
    dots = [float((ref.rope(q, [[[p + 7]]], [4], f, 0) * ref.rope(k, [[[p]]], [4], f, 0)).sum()) for p in (0, 5, 1000)]
    assert np.allclose(dots, dots[0], atol=1e-11)


def test_oracle_keeps_what_the_definition_says():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.2, 0.1]))
    tokens = lambda **kw: np.nonzero(ref.kept(x, **kw))[0].tolist()  # noqa: E731
    assert tokens() == [0, 1, 2, 3, 4]
    assert tokens(top_k=2) == [1, 2] and tokens(top_k=4) == [0, 1, 2, 3]          # equal logits by their ids
    assert tokens(top_p=0.5) == [1, 2] and tokens(top_p=0.0) == [1] and tokens(top_p=0.79) == [1, 2, 3]
    assert tokens(top_k=3, top_p=0.7) == [1, 2] and tokens(min_p=0.4) == [1, 2, 3] and tokens(min_p=2.0) == [1]
    assert ref.sample(x, 0.45)[0] == 1 and ref.sample(x, 0.05)[0] == 0 and ref.sample(x, 0.95)[0] == 4
    assert ref.sample(x, 0.9, temp=0.0)[0] == 1 and ref.sample(x, 1.0)[0] == 4


def test_entry_points_take_no_context():
    L = ema.lib()
    assert L.mgh_sample(None, None, 0, 1, 1, 1, None, None, None, None) == -1
    assert L.mgh_rope(None, None, None, 0, None, 2, 1, 1, 1, None, None, None, None, None) == -1


def test_which_kernels_shared_attention_takes():
    """few rows of a group, 64 and 128 of them to a workgroup; a workgroup of the shared blocks per CU, then the own ones'"""
    run(BODY + """
def call(S, H, Hkv, D, Bn, nb, group, most, **kw):
    kv = ema.Kv8(W, X, B, R, Y, G, nb, 1 << 20, Hkv, D, Bn)
    launches()
    c.kv8_attn_shared(kv, 0x1200000, (1, H * D, D, S * H * D), S, 0x1300000, None, group, 0x1600000, most, H, D ** -0.5, o16=0x1400000, **kw)
    l = launches()
    m = re.search(r"k_kv8_attn_sharedILi(\\d)ELb(\\d)ELb(\\d)ELi(\\d)E", l[0][1])
    return tuple(map(int, m.groups())), l[0][2][0], [k for k, _, _ in l[1:]]

few, many = ["k_attn_join_few"], ["k_attn_join"]
# 256 rows of a key head: two tiles of 128, 16 parts; the own blocks of 64 sequences
assert call(1, 32, 8, 128, 64, 266, 64, 250) == ((4, 0, 0, 2), 8 * 2 * 16 + 512, many)
assert call(1, 32, 8, 128, 64, 266, 16, 250) == ((4, 0, 0, 1), 8 * 4 * 8 + 512, many)
assert call(1, 32, 8, 128, 64, 266, 8, 250) == ((4, 0, 0, 0), 8 * 8 * 2 * 2 + 512, few)
assert call(1, 32, 8, 128, 64, 266, 4, 250)[0] == (4, 0, 0, 0)
# at least eight blocks to a part; no shared block at all
assert call(1, 32, 8, 128, 64, 30, 64, 20) == ((4, 0, 0, 2), 8 * 2 * 3 + 512, few)
assert call(1, 32, 8, 128, 64, 30, 64, 0) == ((4, 0, 0, 2), 8 * 2 + 512, few)
# own rows of more than 16: tiles of 16
assert call(5, 32, 8, 128, 4, 40, 4, 32)[1] == 8 * 4 + 8 * 4 * 2
for D, dg in ((16, 1), (32, 1), (48, 2), (64, 2), (80, 3), (96, 3), (112, 4)):
    assert call(1, 8, 8, D, 64, 8, 64, 4)[0] == (dg, 0, 0, 1)
assert call(1, 8, 8, 64, 64, 8, 64, 4, cap=3.0)[0] == call(1, 8, 8, 64, 64, 8, 64, 4, slopes=0x1500000)[0] == (2, 0, 1, 1)
""")


def test_which_kernels_rope_takes():
    """granules of 4 and 1 pairs by order and alignment; heads of a thread by the number of rows"""
    run(ROPE + """
def call(pairs, D, order=0, in16=True, out16=True, S=9, H=4, Bn=2, x=W, st=None):
    st = st or (1, H * D, D, S * H * D)
    launches()
    c.rope(rot(pairs, order=order), x, st, D, S, H, Bn, in16=in16, y_strides=(1, H * D, D, S * H * D), **{"y16" if out16 else "y": Y})
    (k, n, g), = launches()
    m = re.search(r"k_ropeILi(\\d)ELb(\\d)ELb(\\d)E", n)
    return tuple(map(int, m.groups())), g[:2]

assert call((8,), 16) == ((4, 1, 1), (1, 2))
assert call((8,), 16, in16=False) == ((4, 0, 1), (1, 2)) and call((8,), 16, out16=False)[0] == (4, 1, 0) and call((8,), 16, in16=False, out16=False)[0] == (4, 0, 0)
assert call((12, 12), 48)[0] == (4, 1, 1) and call((12, 12), 48, order=1)[0] == (4, 1, 1) and call((12, 12), 48, order=2)[0] == (4, 1, 1)
assert call((5,), 16)[0] == (1, 1, 1) and call((4,), 16)[0] == (4, 1, 1) and call((0,), 24)[0] == (4, 1, 1) and call((3,), 6)[0] == (1, 1, 1)
assert call((8,), 16, x=W + 2)[0] == (1, 1, 1) and call((8,), 16, x=W + 8)[0] == (4, 1, 1) and call((8,), 16, st=(1, 66, 16, 66 * 9))[0] == (1, 1, 1)
assert call((64,), 128, S=100, H=32)[1] == (100 * 32 * 16 // 256, 2) and call((64,), 128, S=16, H=9)[1] == (16 * 9 * 16 // 256, 2)
assert call((64,), 128, S=65536, H=32)[1] == (65536 * 4 * 16 // 256, 2)
""")


def test_rope_covers_rows_of_every_alignment():
    """threads for all pairs of all heads of all tokens, whatever the rows' and pointers' alignment, of x or y: one, two, four or
    eight elements, with one head of each thread and with several"""
    run(ROPE + """
def call(p, D, S, H, x=W, wx=0, y=Y, wy=0, head=0, seq=0, **kw):
    launches()
    w = H * (D + head)
    out = {"y16" if kw.pop("out16", True) else "y": y}
    c.rope(rot((p,)), x, (1, w + wx, D + head, S * (w + wx) + seq), D, S, H, 2, y_strides=(1, H * D + wy, D, S * (H * D + wy)), **out, **kw)
    (k, n, g), = launches()
    v = int(re.search(r"k_ropeILi(\\d)E", n).group(1))
    return v, g[:2]

for p, D, S, H in ((24, 48, 100, 16), (32, 64, 1000, 32), (8, 16, 9, 4), (12, 48, 33, 5), (0, 32, 70, 3)):
    def needs(v):                                       # heads of a thread: up to 8 while 2^17 threads are left
        n = 1
        while n < 8 and n < H and 2 * S * (D // 2 // v) * H // (2 * n) >= 256 * 512:
            n *= 2
        return v, (-(-S * (D // 2 // v) * -(-H // n) // 256), 2)
    at = lambda **kw: call(p, D, S, H, **kw)  # noqa: E731
    for wide, v in ((0, 4), (1, 1), (2, 1), (3, 1), (4, 4), (6, 1), (8, 4), (10, 1), (12, 4)):
        got = [at(wx=wide), at(wy=wide), at(seq=wide), at(wx=wide, in16=False), at(wy=wide, out16=False), at(head=wide), at(wx=wide, in16=False, out16=False)]
        assert got == [needs(v)] * 7, (wide, got, needs(v))
    for b, v in ((2, 1), (4, 1), (6, 1), (8, 4), (10, 1), (12, 1), (16, 4)):
        assert at(x=W + b) == at(y=Y + b) == needs(v), (b, at(x=W + b), at(y=Y + b), needs(v))
    for b in (4, 8, 12):
        assert at(x=W + b, in16=False) == at(y=Y + b, out16=False) == needs(1), b
""")


def test_which_kernels_sampling_takes():
    """rows up to 2048 and 8192 tokens in one workgroup, longer ones in chunks of 8192, rows by rows of 128 MB"""
    run(BODY + """
def call(rows, V, **kw):
    launches()
    c.sample(W, rows, V, X, Y, **kw)
    return [(k, g[:2]) for k, _, g in launches()]

assert call(3, 2048) == [("k_sample", (3, 1))] and call(3, 2049) == call(3, 8192) == [("k_sample", (3, 1))]
assert call(3, 8193) == [("k_sample_range", (2, 3)), ("k_sample_bins", (2, 3)), ("k_sample_pick", (1, 3))]
l = call(1000, 128001, f16=True)
assert [k for k, _ in l] == ["k_sample_range", "k_sample_bins", "k_sample_pick"] * 3
assert sum(g[1] for k, g in l if k == "k_sample_pick") == 1000
assert call(1, 1 << 24)[0] == ("k_sample_range", (2048, 1))
c.graph_begin()
try:
    call(1, (1 << 24) - 1)
    call(64, 128001)
finally:
    c.graph_end().destroy()
""")


def device_kernels():
    """{name: metadata} of the built library's kernels: the note of each device code object in its bundles"""
    ema.lib()
    with open(os.path.join(os.path.dirname(ema.__file__), "lib", "libmgh.so"), "rb") as f:
        data = f.read()
    magic, found, at = b"__CLANG_OFFLOAD_BUNDLE__", {}, 0
    while (at := data.find(magic, at)) >= 0:
        entry = at + len(magic) + 8
        for _ in range(struct.unpack_from("<Q", data, at + len(magic))[0]):
            off, size, n = struct.unpack_from("<QQQ", data, entry)
            if size and b"gfx950" in data[entry + 24:entry + 24 + n]:
                obj = data[at + off:at + off + size]
                note = obj.find(b"AMDGPU\0\0")
                notes = struct.unpack_from("<III", obj, note - 12)
                for k in msgpack.unpackb(obj[note + 8:note + 8 + notes[1]])["amdhsa.kernels"]:
                    found[k[".name"]] = k
            entry += 24 + n
        at += len(magic)
    return found


def test_cache_attention_keeps_its_registers():
    """no kernel of the cache's attention has scratch memory (a register spilled across its loop cost 3% of capped calls)"""
    attn = {n: k for n, k in device_kernels().items() if "k_kv8_attn" in n}
    assert len(attn) == 32 + 48
    assert [n for n, k in attn.items() if k[".private_segment_fixed_size"]] == []
