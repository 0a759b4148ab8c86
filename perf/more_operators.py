"""What a generating step does beside attention under masks: what the operators compute in plain form, and the
calls that a program makes of the MI355X kernels for them.

Kinds:
  rope    rotary positions with one to three axes (index; row and column; time, row and column) on the heads of
          queries and keys; fp16 or fp32 in and out, whole or part of a head's features, three orders of pairs
  append  new keys, rotated on the way, and values into the 8-bit cache (blocks of 32 tokens, a scale per block and
          head), the rotated queries, and the values that the touched blocks now stand for
  shared  attention of the newest tokens over that cache where groups of sequences share their first blocks
  sample  a token drawn from logits with temperature, top-k, top-p and min-p, from given random numbers

Head layouts are those of this backend's models (16 heads of 48) and generic ones (heads of 64 and 128, grouped by
4); token rows those of 256-, 1024- and 4096-token images with their class token, prompts and contexts of up to
100 thousand tokens. Vocabularies: the model's 2025 and generic ones to 128 thousand.

Everything that a program holds before the call (activations, positions, the cache's pages and its table, output
buffers) is made in prepare().
"""
import math
import random

import torch

own = False

BLOCK, RING = 32, 64          # tokens of a cache block; tokens kept in fp16 behind the last whole block
VOCAB = 2025
HALVES, PAIRS, AXIS_HALVES = 0, 1, 2   # pair i: features (i, P + i); (2 i, 2 i + 1); halves of each axis's own features


def listed():
    return [
        # queries and keys of one image of 16 x 16 tokens and its class token, rows and columns, on the fp32 output
        # of the QKV product: the smallest call, where latency counts
        dict(name="rope_image", kind="rope", batch=1, tokens=257, heads=32, dim=48, pairs="12+12", order=AXIS_HALVES,
             in16=False, out16=True),
        # a long prompt, the first half of each head's features, positions far out
        dict(name="rope_text", kind="rope", batch=3, tokens=1021, heads=40, dim=64, pairs="16", order=PAIRS,
             in16=False, out16=False),
        # two clips of video: time, row and column
        dict(name="rope_video", kind="rope", batch=2, tokens=8191, heads=40, dim=128, pairs="16+24+24", order=HALVES,
             in16=True, out16=True),
        # the queries, keys and values of four prompts of different lengths
        dict(name="append_prompt", kind="append", batch=4, new=2050, past=0, heads=32, kv_heads=8, dim=128, pairs="64",
             order=HALVES, f16=True),
        # one token of each of 64 sequences, some of which complete a block
        dict(name="append_token", kind="append", batch=64, new=1, past=5000, heads=32, kv_heads=8, dim=128, pairs="64",
             order=HALVES, f16=True),
        # images of 32 x 32 tokens behind a text, the model's own heads, fp32 rows
        dict(name="append_image", kind="append", batch=4, new=1025, past=96, heads=16, kv_heads=16, dim=48, pairs="12+12",
             order=AXIS_HALVES, f16=False),
        # one token of each of 64 sequences that go on from one prompt
        dict(name="shared_prompt", kind="shared", batch=64, group=64, new=1, prefix=8000, past=500, heads=32, kv_heads=8,
             dim=128, cap=0.0, slopes=False),
        # eight answers to each of eight questions, capped scores
        dict(name="shared_answers", kind="shared", batch=64, group=8, new=1, prefix=4000, past=700, heads=32, kv_heads=8,
             dim=128, cap=30.0, slopes=False),
        # five drafted tokens of each of four sequences, the model's own heads (no grouping): the smallest
        dict(name="shared_draft", kind="shared", batch=4, group=4, new=5, prefix=1024, past=40, heads=16, kv_heads=16, dim=48,
             cap=0.0, slopes=True),
        # one row of the model's vocabulary: launches count
        dict(name="sample_row", kind="sample", rows=1, vocab=VOCAB, top_k=100, top_p=0.95, min_p=0.0, spread=3.0, f16=False),
        # every position of four images, the whole vocabulary but its unlikely end
        dict(name="sample_grid", kind="sample", rows=1028, vocab=VOCAB, top_k=0, top_p=0.0, min_p=0.02, spread=3.0, f16=False),
        # a batch of rows of a large vocabulary
        dict(name="sample_batch", kind="sample", rows=64, vocab=128001, top_k=50, top_p=0.9, min_p=0.0, spread=2.5, f16=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _axes(case):
    """pairs of each axis"""
    return [int(n) for n in case["pairs"].split("+")]


def _pairs(rng, dim):
    part = rng.choice([dim // 2, dim // 2, dim // 4])
    axes = rng.choice([1, 1, 2, 3])
    if axes == 1:
        return f"{part}"
    if axes == 2:
        return f"{part // 2}+{part - part // 2}"
    return f"{part - 2 * (3 * part // 8)}+{3 * part // 8}+{3 * part // 8}"


def draw(rng):
    kind = rng.choice(["rope", "append", "shared", "shared", "sample", "sample"])
    dim = rng.choice([32, 48, 48, 64, 64, 80, 96, 112, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 4])
    order = rng.choice([HALVES, PAIRS, AXIS_HALVES])
    if kind == "rope":
        tokens = _log_int(rng, 1, 8191)
        heads = _log_int(rng, 1, 40)
        return dict(kind=kind, batch=_log_int(rng, 1, max(1, min(64, 2 * 8191 * 20 * 128 // (tokens * heads * dim)))),
                    tokens=tokens, heads=heads, dim=dim, pairs=_pairs(rng, dim), order=order, in16=rng.random() < 0.6,
                    out16=rng.random() < 0.7)
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, batch=_log_int(rng, 1, 64), new=rng.randint(1, BLOCK), past=_log_int(rng, 1, 5000),
                        heads=min(heads, 32), kv_heads=kv, dim=dim, pairs=_pairs(rng, dim), order=order, f16=rng.random() < 0.7)
        kv = min(kv, 8)
        return dict(kind=kind, batch=rng.randint(1, 4), new=_log_int(rng, 33, 2050), past=rng.choice([0, 96, 1000]),
                    heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=dim, pairs=_pairs(rng, dim), order=order,
                    f16=rng.random() < 0.7)
    if kind == "shared":
        group = _log_int(rng, 1, 64)
        batch = min(64, group * rng.choice([1, 1, 2, 3, 5]) + rng.choice([0, 0, 1]))
        new = rng.choice([1, 1, 1, 2, 5])
        prefix = _log_int(rng, 1, 250) * BLOCK
        past = _log_int(rng, 1, 700)
        return dict(kind=kind, batch=batch, group=group, new=new, prefix=prefix, past=past, heads=min(heads, 32),
                    kv_heads=min(kv, 8) if heads > 32 else kv, dim=dim, cap=rng.choice([0.0, 0.0, 30.0]),
                    slopes=rng.random() < 0.3)
    vocab = _log_int(rng, 100, 128001)
    return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(1028, 64 * 128001 // vocab))), vocab=vocab,
                top_k=rng.choice([0, 1, 50, _log_int(rng, 1, vocab)]), top_p=rng.choice([0.0, 0.5, 0.9, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.05, 0.3]), spread=rng.choice([0.5, 2.5, 4.0]), f16=rng.random() < 0.4)


# ---- inputs -------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6271 + 17)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _freqs(pairs):
    """angle per unit of position of each pair: from 1 down to nearly 1 / 10000 along each axis"""
    return [10000.0 ** (-i / n) for n in pairs for i in range(n)]


def _grid(axes, n, b):
    """positions of the n tokens of sequence b along each of two or three axes, as images and clips are laid out:
    a first token of its own, then rows of a square grid (or of clips of 16 frames)"""
    i = torch.arange(-1, n - 1, device="cuda")
    side = max(1, int(round(math.sqrt(n / (16 if axes == 3 else 1)))))
    at = [i // side % side if axes == 3 else i // side, i % side]
    if axes == 3:
        at = [i // (side * side)] + at
    return torch.stack([torch.where(i < 0, torch.zeros_like(i), x + 1 + b) for x in at])


def _positions(case, n):
    """[axes][B][n] positions, or None: consecutive ones"""
    axes = len(_axes(case))
    if axes == 1:
        return None
    return torch.stack([_grid(axes, n, b) for b in range(case["batch"])], 1).to(torch.int32).contiguous()


def _firsts(case):
    """first positions of consecutive ones: far out for the first sequence"""
    r = random.Random(case["tokens"])
    return [100003] + [r.randint(0, 50000) for _ in range(case["batch"] - 1)]


def _prepare_rope(case, seed):
    g, bt, n, h, d = _gen(seed), *(case[k] for k in ("batch", "tokens", "heads", "dim"))
    w = h * d + 128                       # the rows hold something behind the heads that turn
    dt = [torch.float32, torch.float16]
    s = {"case": case, "x": _randn(g, bt, n, w).to(dt[case["in16"]]), "pos": _positions(case, n), "first": _ints(_firsts(case))}
    s["y"] = torch.zeros(bt, n, h * d, dtype=dt[case["out16"]], device="cuda")
    s["freqs"] = _freqs(_axes(case))
    return s


def _past(case):
    """cached tokens of each sequence before the call: the first has `past`, the others down to 1/16 of it"""
    r = random.Random(case["past"] * 13 + case["batch"])
    lens = [case["past"]] + [int(case["past"] * 16.0 ** -r.random()) for _ in range(case["batch"] - 1)]
    if case["kind"] == "shared":
        return [n + s * BLOCK for n, s in zip(lens, _by_sequence(case))]
    # a prompt's pieces start where a block starts
    return [n // BLOCK * BLOCK for n in lens] if case["new"] > BLOCK else lens


def _new(case):
    """new tokens of each sequence"""
    r = random.Random(case["new"] * 17 + case["batch"])
    return [case["new"]] + [r.randint((case["new"] + 1) // 2, case["new"]) for _ in range(case["batch"] - 1)]


def _shared(case):
    """blocks that each group shares: the first group has the most"""
    r = random.Random(case["prefix"] * 5 + case["group"])
    groups = -(-case["batch"] // case["group"])
    most = case["prefix"] // BLOCK
    return [most] + [r.randint((most + 1) // 2, most) for _ in range(groups - 1)]


def _by_sequence(case):
    sh = _shared(case)
    return [sh[b // case["group"]] for b in range(case["batch"])]


def _to_v_layout(v):
    """codes [pages][heads][32 tokens][D] as the cache keeps V: [pages][heads][D / 2][4][2][8]"""
    p, h, _, d = v.shape
    return v.view(p, h, 4, 8, d // 2, 2).permute(0, 1, 4, 2, 5, 3).contiguous()


def _from_v_layout(v, d):
    p, h = v.shape[:2]
    return v.view(p, h, d // 2, 4, 2, 8).permute(0, 1, 3, 5, 2, 4).reshape(p, h, BLOCK, d)


def _codes(x):
    """Q8 codes + 128 of blocks [pages][heads][32][D] and their scales"""
    d = (x.abs().amax((-1, -2)).double() / 127).float()
    return (x / d[:, :, None, None]).round().clamp(-127, 127).add(128).to(torch.uint8), d


def _tables(case, lens, new, seed):
    """pages of each sequence's blocks, in any order; the blocks that a group shares are the same pages"""
    used = [-(-(n + m) // BLOCK) for n, m in zip(lens, new)]
    same = _by_sequence(case) if case["kind"] == "shared" else [0] * len(lens)
    total = sum(u - s for u, s in zip(used, same)) + (sum(_shared(case)) if case["kind"] == "shared" else 0)
    pages, nb = total + 2, max(used)
    perm = list(range(pages))
    random.Random(seed).shuffle(perm)
    table, common = [], []
    for b, u in enumerate(used):
        if case["kind"] == "shared" and b % case["group"] == 0:
            common = [perm.pop() for _ in range(same[b])]
        table.append(common + [perm.pop() for _ in range(u - same[b])] + [-1] * (nb - u))
    return pages, nb, table


def _prepare_cache(case, seed):
    """the cache with every token up to lens + new in it ("shared") or up to lens ("append")"""
    g, bt, h, hk, d = _gen(seed), *(case[k] for k in ("batch", "heads", "kv_heads", "dim"))
    lens, new = _past(case), _new(case)
    pages, nb, table = _tables(case, lens, new, seed)
    s = {"case": case, "pages": pages, "blocks": nb, "lens": _ints(lens), "new": _ints(new), "table": _ints(table)}
    s["k_tail"], s["v_tail"] = _randn(g, bt, hk, RING, d).half(), _randn(g, bt, hk, d, RING).half()
    if case["kind"] == "shared":
        spread = torch.exp(0.5 * _randn(g, 1, hk, 1, d))         # some features are larger than others
        k, dk = _codes((_randn(g, pages, hk, BLOCK, d) * spread).half().float())
        v, dv = _codes(_randn(g, pages, hk, BLOCK, d).half().float())
        s["k"], s["v"], s["scales"] = k, _to_v_layout(v), torch.stack((dk, dv), -1).contiguous()
        s["shared"] = _ints(_shared(case))
        s["q"] = (2 * _randn(g, bt, case["new"], h * d)).half()
        s["o"] = torch.zeros_like(s["q"])
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slopes"] else None
        return s
    s["k"] = torch.full((pages, hk, BLOCK, d), 128, dtype=torch.uint8, device="cuda")
    s["v"] = torch.full((pages, hk, d // 2, 4, 2, 8), 128, dtype=torch.uint8, device="cuda")
    s["scales"] = torch.zeros(pages, hk, 2, device="cuda")
    rows = _randn(g, bt, case["new"], (h + 2 * hk) * d)           # the fused QKV product's rows
    s["rows"] = rows.half() if case["f16"] else rows
    s["pos"], s["freqs"] = _positions(case, case["new"]), _freqs(_axes(case))
    s["q"] = torch.zeros(bt, case["new"], h * d, dtype=torch.float16, device="cuda")
    first = [n // BLOCK * BLOCK for n in lens]
    s["first"], s["total"] = _ints(first), _ints([n + m for n, m in zip(lens, new)])
    s["span"] = max(n + m - f for n, m, f in zip(lens, new, first))
    s["out"] = [torch.zeros(bt, hk, s["span"], d, dtype=torch.float16, device="cuda") for _ in range(2)]
    return s


def _prepare_sample(case, seed):
    g, rows, vocab = _gen(seed), case["rows"], case["vocab"]
    x = case["spread"] * _randn(g, rows, vocab)
    x = torch.where(torch.rand(rows, vocab, generator=g, device="cuda") < 0.02, x * 1.5, x)     # a few stand out
    s = {"case": case, "x": x.half() if case["f16"] else x}
    # what each request asked for; one in sixteen wants the most likely token
    s["temp"] = 0.6 + 0.8 * torch.rand(rows, generator=g, device="cuda")
    s["temp"][5::16] = 0
    r = random.Random(seed)
    if case["top_k"]:
        s["top_k"] = _ints([case["top_k"]] + [r.randint((case["top_k"] + 1) // 2, case["top_k"]) for _ in range(rows - 1)])
    if case["top_p"]:
        s["top_p"] = torch.tensor([case["top_p"]] + [case["top_p"] * r.uniform(0.9, 1) for _ in range(rows - 1)], device="cuda")
    if case["min_p"]:
        s["min_p"] = torch.tensor([case["min_p"]] + [case["min_p"] * r.uniform(0.5, 1) for _ in range(rows - 1)], device="cuda")
    s["u"] = torch.rand(rows, generator=g, device="cuda")
    s["ids"], s["prob"] = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    return s


def prepare(case, seed):
    s = {"rope": _prepare_rope, "append": _prepare_cache, "shared": _prepare_cache, "sample": _prepare_sample}[case["kind"]](case, seed)
    # device addresses, as a program that binds the C ABI holds them
    s["ptr"] = {k: v.data_ptr() for k, v in s.items() if torch.is_tensor(v)}
    return s


# ---- plain forms ----------------------------------------------------------------------------


def _features(case):
    """the two features of each pair"""
    pairs, order = _axes(case), case["order"]
    if order == PAIRS:
        lo = [2 * i for i in range(sum(pairs))]
        return lo, [x + 1 for x in lo]
    if order == HALVES:
        lo = list(range(sum(pairs)))
        return lo, [x + sum(pairs) for x in lo]
    lo, hi, at = [], [], 0
    for n in pairs:
        lo += range(at, at + n)
        hi += range(at + n, at + 2 * n)
        at += 2 * n
    return lo, hi


def _turn(x, pos, case, freqs):
    """x [B,S,H,D] in 64 bits, pos [axes][B][S]; angles of far positions need 64 bits, and so does a value that
    is rounded to fp16 and then to a code"""
    axis = torch.tensor([a for a, n in enumerate(_axes(case)) for _ in range(n)], device="cuda")
    ang = pos.double().permute(1, 2, 0)[:, :, axis] * torch.tensor(freqs, dtype=torch.float64, device="cuda")
    c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
    lo, hi = _features(case)
    a, b = x[..., lo], x[..., hi]
    y = x.clone()
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    return y


def _run_of(first, n, axes):
    """consecutive positions along every axis"""
    return (first[:, None].long() + torch.arange(n, device="cuda")).expand(axes, -1, -1)


def _plain_rope(s):
    case = s["case"]
    bt, n, h, d = (case[k] for k in ("batch", "tokens", "heads", "dim"))
    x = s["x"][:, :, :h * d].reshape(bt, n, h, d).float()
    pos = _run_of(s["first"], n, 1) if s["pos"] is None else s["pos"]
    axis = torch.tensor([a for a, m in enumerate(_axes(case)) for _ in range(m)], device="cuda")
    ang = pos.double().permute(1, 2, 0)[:, :, axis] * torch.tensor(s["freqs"], dtype=torch.float64, device="cuda")
    c, si = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]
    lo, hi = _features(case)
    a, b = x[..., lo], x[..., hi]
    y = x.clone()
    y[..., lo], y[..., hi] = a * c - b * si, a * si + b * c
    return y.reshape(bt, n, h * d).to(s["y"].dtype)


def _ring(s, pos):
    """k, v [B,Hk,n,D] of the fp16 ring at positions pos [B,n]"""
    bt, hk, d = (s["case"][k] for k in ("batch", "kv_heads", "dim"))
    slot = (pos % RING)[:, None, :, None].expand(bt, hk, pos.shape[1], d)
    return s["k_tail"].gather(2, slot), s["v_tail"].transpose(2, 3).gather(2, slot)


def _plain_append(s):
    case = s["case"]
    bt, h, hk, d, n = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "new"))
    pos = _run_of(s["lens"], n, len(_axes(case))) if s["pos"] is None else s["pos"]
    rows = s["rows"].view(bt, n, h + 2 * hk, d)
    turned = _turn(rows[:, :, :h + hk].double(), pos, case, s["freqs"]).half()
    mine = torch.arange(n, device="cuda")[None, :] < s["new"][:, None]      # a sequence's own rows
    q = torch.where(mine[:, :, None], turned[:, :, :h].reshape(bt, n, h * d), torch.zeros_like(s["q"]))
    span = -(-s["span"] // BLOCK) * BLOCK
    at_pos = s["first"][:, None].long() + torch.arange(span, device="cuda")
    at = at_pos - s["lens"][:, None]                                # index among the new tokens
    here = (at_pos < s["total"][:, None])[:, None, :, None]
    pick = at.clamp(0, n - 1)[:, None, :, None].expand(bt, hk, span, d)
    whole = ((s["first"][:, None] + torch.arange(BLOCK, span + 1, BLOCK, device="cuda")) <= s["total"][:, None])
    out = [q]
    for kv, old in zip((turned[:, :, h:], rows[:, :, h + hk:].half()), _ring(s, at_pos)):
        raw = torch.where((at < 0)[:, None, :, None], old, kv.transpose(1, 2).gather(2, pick))
        y = torch.where(here, raw, torch.zeros_like(raw)).view(bt, hk, span // BLOCK, BLOCK, d)
        scale = (y.abs().amax((-1, -2)).double() / 127).float()[..., None, None]
        t = y.double() / scale                       # next to a border 32 bits would take the other code
        code = torch.sign(t) * torch.floor(t.abs() + 0.5)
        val = torch.where(scale > 0, code, torch.zeros_like(code)).float() * scale
        val = torch.where(whole[:, None, :, None, None], val, y.float()).view(bt, hk, span, d)
        out.append(torch.where(here, val, torch.zeros_like(val))[:, :, :s["span"]].half())
    return out


def _plain_shared(s):
    case = s["case"]
    bt, n, h, hk, d = (case[k] for k in ("batch", "new", "heads", "kv_heads", "dim"))
    out = torch.zeros(bt, n, h, d, dtype=torch.float16, device="cuda")
    for b0 in range(0, bt, 8):                       # (eight sequences' scores at a time)
        b1 = min(bt, b0 + 8)
        total = (s["lens"][b0:b1] + s["new"][b0:b1])[:, None]
        keys = torch.arange(s["blocks"] * BLOCK, device="cuda")
        pages = s["table"][b0:b1].clamp(min=0).long()
        kv = []
        for codes, i in ((s["k"], 0), (_from_v_layout(s["v"], d), 1)):
            x = (codes[pages].float() - 128) * s["scales"][pages][..., i][..., None, None]
            kv.append(x.transpose(1, 2).reshape(b1 - b0, hk, -1, d))
        slot = (keys % RING)[None, None, :, None].expand(b1 - b0, hk, -1, d)
        raw = (keys[None] >= total // BLOCK * BLOCK)[:, None, :, None]
        live = (keys[None] < total)[:, None, :, None]
        k = torch.where(raw, s["k_tail"][b0:b1].gather(2, slot).float(), kv[0]).masked_fill(~live, 0)
        v = torch.where(raw, s["v_tail"][b0:b1].transpose(2, 3).gather(2, slot).float(), kv[1]).masked_fill(~live, 0)
        pos = (s["lens"][b0:b1, None] + torch.arange(n, device="cuda"))[:, None, None, :, None]
        q = s["q"][b0:b1].float().view(b1 - b0, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b1 - b0, hk, -1, d)
        sc = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b1 - b0, hk, h // hk, n, -1) * d ** -0.5
        if case["cap"]:
            sc = (sc / case["cap"]).tanh() * case["cap"]
        if s["slopes"] is not None:
            sc = sc - s["slopes"].view(1, hk, h // hk, 1, 1) * (pos - keys).abs()
        sc = sc.masked_fill(keys > pos, -math.inf).view(b1 - b0, hk, -1, len(keys))
        p = (sc - sc.amax(-1, keepdim=True)).exp()
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[b0:b1] = o.view(b1 - b0, hk, h // hk, n, d).permute(0, 3, 1, 2, 4).reshape(b1 - b0, n, h, d).half()
    mine = torch.arange(n, device="cuda")[None, :] < s["new"][:, None]  # a sequence's own rows; the others stay as they were
    return torch.where(mine[:, :, None, None], out, torch.zeros_like(out)).view(bt, n, h * d)


def _plain_sample(s):
    """in 64 bits: what lies next to the border of a running sum decides which token it is"""
    case, x = s["case"], s["x"].double()
    rows, vocab = x.shape
    rank = torch.arange(vocab, device="cuda")
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = s["temp"].double()[:, None]
    greedy = t <= 0
    w = ((top - top[:, :1]) / torch.where(greedy, torch.ones_like(t), t)).exp()
    keep = (rank < s["top_k"][:, None]) if case["top_k"] else torch.ones_like(w, dtype=torch.bool)
    if case["top_p"]:
        mass = (w * keep).cumsum(1)
        keep = keep & (mass - w < s["top_p"].double()[:, None] * mass[:, -1:])
    if case["min_p"]:
        keep = keep & (w >= s["min_p"].double()[:, None])
    keep = torch.where(greedy, rank[None] == 0, keep)
    w = torch.zeros_like(w).scatter_(1, order, w * keep)            # back to the order of the ids
    mass = w.cumsum(1)
    total = mass[:, -1:]
    ids = (mass <= s["u"].double()[:, None] * total).sum(1).clamp(max=vocab - 1)
    return [ids.to(torch.int32), (w.gather(1, ids[:, None]) / total)[:, 0].float()]


# ---- the framework's calls --------------------------------------------------------------------

_CTX = []


def _ctx():
    """the program's one kernel context"""
    if not _CTX:
        import edge_maskgit_amd as ema
        _CTX.append(ema.Context(0))
    return _CTX[0]


def _rope(s, n):
    """the rotation, which a program keeps with its positions"""
    if "rope" not in s:
        import edge_maskgit_amd as ema
        case = s["case"]
        s["rope"] = ema.Rope(_axes(case), s["freqs"], case["order"], s["ptr"].get("pos"), (1, n, case["batch"] * n))
    return s["rope"]


def _own_rope(s):
    case, p = s["case"], s["ptr"]
    bt, n, h, d = (case[k] for k in ("batch", "tokens", "heads", "dim"))
    w = h * d + 128
    _ctx().rope(_rope(s, n), p["x"], (1, w, d, n * w), d, n, h, bt, in16=case["in16"], first=p["first"],
                y_strides=(1, h * d, d, n * h * d), **{"y16" if case["out16"] else "y": p["y"]})
    return s["y"]


def _handle(s):
    """the cache's handle, which a program keeps with its buffers"""
    if "handle" not in s:
        import edge_maskgit_amd as ema
        case, p = s["case"], s["ptr"]
        s["handle"] = ema.Kv8(p["k"], p["v"], p["scales"], p["k_tail"], p["v_tail"], p["table"], s["blocks"], s["pages"],
                              case["kv_heads"], case["dim"], case["batch"])
    return s["handle"]


def _own_append(s):
    case, p, c, kv8 = s["case"], s["ptr"], _ctx(), _handle(s)
    h, hk, d, n = case["heads"], case["kv_heads"], case["dim"], case["new"]
    w, e = (h + 2 * hk) * d, 2 if case["f16"] else 4
    st = (1, w, d, n * w)
    c.kv8_append_rope(kv8, _rope(s, n), p["rows"] + e * h * d, p["rows"] + e * (h + hk) * d, st, n, p["lens"], p["new"],
                      in16=case["f16"], q=p["rows"], q_strides=st, H=h, q_out=p["q"], qo_strides=(1, h * d, d, n * h * d))
    c.kv8_read(kv8, p["first"], s["span"], p["total"], k16=s["out"][0].data_ptr(), v16=s["out"][1].data_ptr())
    return [s["q"]] + s["out"]


def _own_shared(s):
    case, p = s["case"], s["ptr"]
    n, h, d = case["new"], case["heads"], case["dim"]
    st = (1, h * d, d, n * h * d)
    _ctx().kv8_attn_shared(_handle(s), p["q"], st, n, p["lens"], p["new"], case["group"], p["shared"], case["prefix"] // BLOCK, h,
                           d ** -0.5, in16=True, cap=case["cap"], slopes=p.get("slopes"), o16=p["o"], o_strides=st)
    return s["o"]


def _own_sample(s):
    case, p = s["case"], s["ptr"]
    _ctx().sample(p["x"], case["rows"], case["vocab"], p["u"], p["ids"], f16=case["f16"], temp=p["temp"], top_k=p.get("top_k"),
                  top_p=p.get("top_p"), min_p=p.get("min_p"), prob=p["prob"])
    return [s["ids"], s["prob"]]


def run(state):
    kind = state["case"]["kind"]
    if kind == "rope":
        return _own_rope(state) if own else _plain_rope(state)
    if kind == "append":
        return _own_append(state) if own else _plain_append(state)
    if kind == "shared":
        return _own_shared(state) if own else _plain_shared(state)
    return _own_sample(state) if own else _plain_sample(state)


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    if case["kind"] == "rope":
        n = case["batch"] * case["tokens"]
        by = n * case["heads"] * case["dim"] * ((2 if case["in16"] else 4) + (2 if case["out16"] else 4))
        pos = 4 * n * len(_axes(case)) if len(_axes(case)) > 1 else 4 * case["batch"]
        return {"bytes": by + pos, "flops": 6 * n * case["heads"] * sum(_axes(case))}
    if case["kind"] == "append":
        # new tokens in, rotated queries and codes (or fp16) out; then the touched blocks' codes in, their values out
        h, hk, d, e = case["heads"], case["kv_heads"], case["dim"], 2 if case["f16"] else 4
        n, span = sum(_new(case)), sum(m + t % BLOCK for t, m in zip(_past(case), _new(case)))
        return {"bytes": n * h * d * (e + 2) + 2 * hk * d * (n * e + span * (1 + 1 + 2)),
                "flops": 6 * n * (h + hk) * sum(_axes(case)) + 2 * hk * d * 4 * span}
    if case["kind"] == "shared":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        total = [t + m for t, m in zip(_past(case), _new(case))]
        mine = [t - s * BLOCK for t, s in zip(total, _by_sequence(case))]
        sh = sum(_shared(case))
        by = sum(2 * hk * d * (t + t % BLOCK) + 8 * hk * (t // BLOCK) + 4 * -(-t // BLOCK) for t in mine)
        by += sh * (2 * hk * d * BLOCK + 8 * hk + 4)
        return {"bytes": by + 4 * h * d * sum(_new(case)), "flops": sum(4 * d * h * t * m for t, m in zip(total, _new(case)))}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (2 if case["f16"] else 4) + 28 * case["rows"], "flops": 4 * n}


# ---- the definition in 64 bits ---------------------------------------------------------------


def _angles64(case, seqs, n):
    """cos and sin [axes' pairs][S] of a sequence's positions [axes][S]"""
    out, i = [], 0
    for a, m in enumerate(_axes(case)):
        for j in range(m):
            out.append(seqs[a].double() * 10000.0 ** (-j / m))
            i += 1
    t = torch.stack(out)
    return torch.cos(t), torch.sin(t)


def _turned64(case, x, pos):
    """x [S,H,D] in 64 bits, one pair of features after another"""
    cos, sin = _angles64(case, pos, x.shape[0])
    y, i, base, total = x.clone(), 0, 0, sum(_axes(case))
    for m in _axes(case):
        for j in range(m):
            f, g = {PAIRS: (2 * i, 2 * i + 1), HALVES: (i, i + total), AXIS_HALVES: (base + j, base + m + j)}[case["order"]]
            c, s = cos[i][:, None], sin[i][:, None]
            y[:, :, f] = x[:, :, f] * c - x[:, :, g] * s
            y[:, :, g] = x[:, :, f] * s + x[:, :, g] * c
            i += 1
        base += 2 * m
    return y


def _pos64(case, s, b, n, start):
    if s["pos"] is None:
        return [torch.arange(start, start + n, device="cuda")]
    return [s["pos"][a, b, :n] for a in range(len(_axes(case)))]


def _exact_rope(case, s):
    bt, n, h, d = (case[k] for k in ("batch", "tokens", "heads", "dim"))
    out = torch.empty(bt, n, h * d, dtype=torch.float64, device="cuda")
    for b in range(bt):
        x = s["x"][b, :, :h * d].double().view(n, h, d)
        out[b] = _turned64(case, x, _pos64(case, s, b, n, _firsts(case)[b])).view(n, h * d)
    return out


def _exact_append(case, s):
    h, hk, d, n = case["heads"], case["kv_heads"], case["dim"], case["new"]
    q = torch.zeros(case["batch"], n, h * d, dtype=torch.float64, device="cuda")
    outs = [torch.zeros(case["batch"], hk, s["span"], d, dtype=torch.float64, device="cuda") for _ in range(2)]
    for b, (past, m) in enumerate(zip(_past(case), _new(case))):
        x = s["rows"][b, :m].double().view(m, h + 2 * hk, d)
        y = _turned64(case, x[:, :h + hk], _pos64(case, s, b, m, past))
        q[b, :m] = y[:, :h].reshape(m, h * d)
        lo = past // BLOCK * BLOCK
        slots = torch.arange(lo, past, device="cuda") % RING
        for which, new in enumerate((y[:, h:].half(), x[:, h + hk:].half())):
            tail = s["k_tail"][b][:, slots] if which == 0 else s["v_tail"][b][:, :, slots].transpose(1, 2)
            t = torch.cat((tail.double(), new.double().transpose(0, 1)), 1)               # [Hk][tokens][D]
            for i in range(0, (past + m - lo) // BLOCK * BLOCK, BLOCK):
                blk = t[:, i:i + BLOCK]
                unit = (blk.abs().flatten(1).max(1).values / 127).float().double()[:, None, None]
                near = torch.trunc(blk / unit)
                near = near + torch.sign(blk) * ((blk / unit - near).abs() >= 0.5)
                t[:, i:i + BLOCK] = torch.where(unit > 0, near * unit, torch.zeros_like(blk))
            outs[which][b, :, :t.shape[1]] = t
    return [q] + outs


def _token_values(s, table, b, n, have):
    """k, v [Hk,n,D] in 64 bits of the first n tokens of `table`'s blocks, of which `have` are there"""
    d, cut = s["case"]["dim"], have // BLOCK * BLOCK
    t = torch.arange(n, device="cuda")
    page, tok, ring, f = table.long()[t // BLOCK].clamp(min=0), t % BLOCK, t % RING, torch.arange(d, device="cuda")
    kc = s["k"][page, :, tok].double() - 128                                             # [n][Hk][D]
    vc = s["v"].view(s["pages"], -1, d * BLOCK)[page]                                     # [n][Hk][D * 32]
    at = ((f[None, :] // 2) * 4 + tok[:, None] // 8) * 16 + (f[None, :] % 2) * 8 + tok[:, None] % 8
    vc = vc.gather(2, at[:, None, :].expand(-1, vc.shape[1], -1)).double() - 128
    sc = s["scales"][page].double()                                                       # [n][Hk][2]
    old = (t < cut)[:, None, None]
    k = torch.where(old, kc * sc[..., :1], s["k_tail"][b][:, ring].transpose(0, 1).double())
    v = torch.where(old, vc * sc[..., 1:], s["v_tail"][b][:, :, ring].permute(2, 0, 1).double())
    return k.transpose(0, 1), v.transpose(0, 1)


def _long_values(s, b, n):
    """_token_values of a sequence, 4096 tokens at a time (each gathers the 32 tokens of its block)"""
    ks, vs = [], []
    for t0 in range(0, n, 4096):
        k, v = _token_values(s, s["table"][b, t0 // BLOCK:(t0 + 4096) // BLOCK], b, min(4096, n - t0), n - t0)
        ks.append(k)
        vs.append(v)
    return torch.cat(ks, 1), torch.cat(vs, 1)


def _exact_shared(case, s):
    n, h, hk, d = (case[k] for k in ("new", "heads", "kv_heads", "dim"))
    out = torch.zeros(case["batch"], n, h, d, dtype=torch.float64, device="cuda")
    for b, (past, m) in enumerate(zip(_past(case), _new(case))):
        k, v = _long_values(s, b, past + m)
        p, j = past + torch.arange(m, device="cuda")[:, None], torch.arange(past + m, device="cuda")[None, :]
        for i in range(h):
            a = i // (h // hk)
            t = (s["q"][b, :m, i * d:(i + 1) * d].double() @ k[a].t().contiguous()) * d ** -0.5
            if case["cap"]:
                t = case["cap"] * torch.tanh(t / case["cap"])
            if case["slopes"]:
                t = t - float(torch.tensor(2.0 ** (-8.0 * (i + 1) / h), dtype=torch.float32)) * (p - j).abs()
            w = torch.softmax(torch.where(j <= p, t, torch.full_like(t, -math.inf)), -1)
            out[b, :m, i] = w @ v[a]
    return out.reshape(case["batch"], n, h * d)


def _exact_sample(case, s):
    """row by row: the tokens sorted on their own, the ones kept counted, the draw by bisection"""
    ids = torch.zeros(case["rows"], dtype=torch.int32, device="cuda")
    prob = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    for r in range(case["rows"]):
        x, t = s["x"][r].double(), float(s["temp"][r])
        if t <= 0:
            ids[r] = int((x == x.max()).nonzero()[0, 0])
            prob[r] = 1.0
            continue
        order = torch.argsort(-x, stable=True)
        w = torch.exp((x[order] - x[order[0]]) / t)
        n = min(int(s["top_k"][r]), len(w)) if case["top_k"] else len(w)
        run = torch.cumsum(w[:n], 0)
        if case["top_p"]:
            n = min(n, 1 + int((run[:-1] < float(s["top_p"][r]) * run[-1]).sum()))
        if case["min_p"]:
            n = min(n, int((w >= float(s["min_p"][r])).sum()))
        kept, back = torch.sort(order[:n])
        run = torch.cumsum(w[:n][back], 0)
        i = min(n - 1, int(torch.searchsorted(run, float(s["u"][r]) * run[-1], right=True)))
        ids[r] = kept[i].to(torch.int32)
        prob[r] = w[:n][back][i] / run[-1]
    return [ids, prob]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "shared": _exact_shared, "sample": _exact_sample}[case["kind"]](case, s)
