"""The operators of token-by-token generation: what they compute in plain form, and the calls that a
program makes of the MI355X kernels for them.

Kinds:
  attn    attention under a causal, prefix or document mask, with scores capped by a tanh or lowered
          with the distance; grouped heads; fp16 or fp32 in and out
  append  new keys and values into the 8-bit cache (blocks of 32 tokens, a scale per block and head),
          and the values that the touched blocks now stand for
  cache   attention of the newest tokens over that cache
  logits  penalties for repeated tokens, biases and a grammar mask on logits

Head layouts are those of this backend's models (16 heads of 48) and generic ones (heads of 64 and 128,
grouped by 4); token rows those of 256-, 1024- and 4096-token images with their class token, prompts and
contexts of up to 100 thousand tokens. Vocabularies: the model's 2025 and generic ones to 128 thousand.

Everything that a program holds before the call (activations, the cache's pages and its table, output
buffers) is made in prepare().
"""
import math
import random

import torch

own = False

BLOCK, RING = 32, 64          # tokens of a cache block; tokens kept in fp16 behind the last whole block
VOCAB = 2025


def listed():
    return [
        # one image of 256 tokens and its class token, scores lowered with the distance, on the fp32 output
        # of the QKV product: the smallest call of a forward, where latency counts
        dict(name="attn_image", kind="attn", batch=1, sq=257, sk=257, heads=16, kv_heads=16, dim=48, causal=False,
             prefix=0, docs=0, cap=0.0, slopes=True, f16=False),
        # images of different sizes packed into one row of tokens, each attending to itself
        dict(name="attn_packed", kind="attn", batch=2, sq=4097, sk=4097, heads=16, kv_heads=16, dim=64, causal=False,
             prefix=0, docs=9, cap=0.0, slopes=False, f16=True),
        # a long prompt whose first tokens see one another, capped scores, grouped heads: the largest
        dict(name="attn_prefix", kind="attn", batch=1, sq=8191, sk=8191, heads=32, kv_heads=8, dim=128, causal=True,
             prefix=1000, docs=0, cap=50.0, slopes=False, f16=True),
        # the next piece of two prompts against everything before it
        dict(name="attn_piece", kind="attn", batch=2, sq=512, sk=12345, heads=32, kv_heads=8, dim=128, causal=True,
             prefix=0, docs=0, cap=0.0, slopes=False, f16=True),
        # one new token of each sequence over keys kept in fp16
        dict(name="attn_token", kind="attn", batch=8, sq=1, sk=8000, heads=32, kv_heads=8, dim=128, causal=True,
             prefix=0, docs=0, cap=0.0, slopes=True, f16=True),
        # the keys and values of four prompts of different lengths
        dict(name="append_prompt", kind="append", batch=4, new=2050, past=0, kv_heads=8, dim=128, f16=True),
        # one token of each of 64 sequences, some of which complete a block
        dict(name="append_token", kind="append", batch=64, new=1, past=5000, kv_heads=8, dim=128, f16=True),
        # one token of one sequence with a long context: one row of queries, work split over the keys
        dict(name="cache_long", kind="cache", batch=1, new=1, past=99990, heads=32, kv_heads=8, dim=128, cap=0.0,
             slopes=False),
        # one token of each of 64 sequences of very different lengths
        dict(name="cache_batch", kind="cache", batch=64, new=1, past=8000, heads=32, kv_heads=8, dim=128, cap=30.0,
             slopes=False),
        # five drafted tokens to be checked at once, the model's own heads (no grouping)
        dict(name="cache_draft", kind="cache", batch=4, new=5, past=1025, heads=16, kv_heads=16, dim=48, cap=0.0,
             slopes=True),
        # one row of the model's vocabulary: launches count
        dict(name="logits_row", kind="logits", rows=1, vocab=VOCAB, hist=257, bias="shared", mask=True, f16=False),
        # a batch of rows of a large vocabulary with a long history and a mask of its own each
        dict(name="logits_batch", kind="logits", rows=64, vocab=128001, hist=4000, bias="shared", mask=True, f16=False),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    dim = rng.choice([16, 32, 48, 48, 64, 64, 80, 96, 112, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    return dim, kv * rng.choice([1, 1, 2, 3, 4, 4, 8]), kv


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "append", "cache", "cache", "logits"])
    if kind == "attn":
        dim, heads, kv = _heads(rng)
        heads, kv = (heads, kv) if heads <= 32 else (32, 8)
        sk = _log_int(rng, 1, 8191)
        sq = sk if rng.random() < 0.6 else _log_int(rng, 1, min(sk, 1024))
        causal = rng.random() < 0.6
        most = max(1, min(16, 32 * 8191 * 8191 // (sq * sk * heads * 2)))
        return dict(kind=kind, batch=_log_int(rng, 1, most), sq=sq, sk=sk, heads=heads, kv_heads=kv, dim=dim,
                    causal=causal, prefix=rng.choice([0, _log_int(rng, 1, sk)]) if causal else 0,
                    docs=rng.choice([0, _log_int(rng, 1, 20)]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                    slopes=rng.random() < 0.4, f16=rng.random() < 0.7)
    if kind == "append":
        dim, _, kv = _heads(rng)
        if rng.random() < 0.5:
            return dict(kind=kind, batch=_log_int(rng, 1, 64), new=rng.randint(1, BLOCK), past=_log_int(rng, 1, 5000),
                        kv_heads=kv, dim=dim, f16=rng.random() < 0.7)
        return dict(kind=kind, batch=rng.randint(1, 4), new=_log_int(rng, 33, 2050), past=rng.choice([0, 96, 1000]),
                    kv_heads=min(kv, 8), dim=dim, f16=rng.random() < 0.7)
    if kind == "cache":
        dim, heads, kv = _heads(rng)
        past = _log_int(rng, 1, 50000)
        most = max(1, min(64, 64 * 8000 * 8 * 128 // (past * kv * dim)))
        return dict(kind=kind, batch=_log_int(rng, 1, most), new=rng.choice([1, 1, 1, 2, 5, 8]), past=past, heads=heads,
                    kv_heads=kv, dim=dim, cap=rng.choice([0.0, 0.0, 30.0]), slopes=rng.random() < 0.3)
    return dict(kind=kind, rows=_log_int(rng, 1, 64), vocab=_log_int(rng, 100, 128001), hist=rng.choice([0, _log_int(rng, 1, 8000)]),
                bias=rng.choice(["none", "shared", "row"]), mask=rng.random() < 0.6, f16=rng.random() < 0.4)


# ---- inputs -------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 31)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _doc_ids(case):
    """[batch][sk]: documents one after the other, lengths spread widely, a few padding tokens (-1)"""
    rows = []
    for b in range(case["batch"]):
        r = random.Random(case["sk"] * 31 + case["docs"] * 7 + b)
        room = case["sk"] - case["sk"] // 60
        cuts = sorted(r.randint(0, room) for _ in range(case["docs"] - 1))
        ids = []
        for k, (lo, hi) in enumerate(zip([0] + cuts, cuts + [room])):
            ids += [k] * (hi - lo)
        rows.append(ids + [-1] * (case["sk"] - room))
    return rows


def _prefixes(case):
    return [case["prefix"] * (b + 1) // case["batch"] for b in range(case["batch"])]


def _past(case):
    """cached tokens of each sequence before the call: the first has `past`, the others down to 1/16 of it"""
    r = random.Random(case["past"] * 13 + case["batch"])
    lens = [case["past"]] + [int(case["past"] * 16.0 ** -r.random()) for _ in range(case["batch"] - 1)]
    # a prompt's pieces start where a block starts
    return [n // BLOCK * BLOCK for n in lens] if case["kind"] == "append" and case["new"] > BLOCK else lens


def _new(case):
    """new tokens of each sequence"""
    r = random.Random(case["new"] * 17 + case["batch"])
    return [case["new"]] + [r.randint((case["new"] + 1) // 2, case["new"]) for _ in range(case["batch"] - 1)]


def _prepare_attn(case, seed):
    g, bt, sq, sk, h, hk, d = _gen(seed), *(case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    dt = torch.float16 if case["f16"] else torch.float32
    s = {"case": case}
    if sq == sk:                     # the fused QKV product's rows
        w = (h + 2 * hk) * d
        rows = _randn(g, bt, sq, w)
        rows[:, :, :h * d] *= 2
        rows = rows.to(dt)
        s["rows"], s["at"] = rows, (0, h * d, (h + hk) * d)
        s["q_st"] = s["kv_st"] = (1, w, d, sq * w)
    else:
        s["q"], s["kv"] = (2 * _randn(g, bt, sq, h * d)).to(dt), _randn(g, bt, sk, 2 * hk * d).to(dt)
        s["at"] = (0, 0, hk * d)
        s["q_st"], s["kv_st"] = (1, h * d, d, sq * h * d), (1, 2 * hk * d, d, sk * 2 * hk * d)
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slopes"] else None
    s["prefix"] = _ints(_prefixes(case)) if case["prefix"] else None
    s["docs"] = _ints(_doc_ids(case)) if case["docs"] else None
    s["o"] = torch.zeros(bt, sq, h * d, dtype=dt, device="cuda")
    return s


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


def _prepare_cache(case, seed):
    """the cache with every token up to lens + new in it ("cache") or up to lens ("append")"""
    g, bt, hk, d = _gen(seed), *(case[k] for k in ("batch", "kv_heads", "dim"))
    lens, new = _past(case), _new(case)
    nb = max(-(-(n + m) // BLOCK) for n, m in zip(lens, new))
    used = [-(-(n + m) // BLOCK) for n, m in zip(lens, new)]
    pages = sum(used) + 2
    perm = list(range(pages))
    random.Random(seed).shuffle(perm)
    table, at = [], 0
    for u in used:
        table.append(perm[at:at + u] + [-1] * (nb - u))
        at += u
    s = {"case": case, "pages": pages, "blocks": nb, "lens": _ints(lens), "new": _ints(new), "table": _ints(table)}
    if case["kind"] == "cache":
        spread = torch.exp(0.5 * _randn(g, 1, hk, 1, d))         # some features are larger than others
        k, dk = _codes((_randn(g, pages, hk, BLOCK, d) * spread).half().float())
        v, dv = _codes(_randn(g, pages, hk, BLOCK, d).half().float())
        s["k"], s["v"], s["scales"] = k, _to_v_layout(v), torch.stack((dk, dv), -1).contiguous()
    else:
        s["k"] = torch.full((pages, hk, BLOCK, d), 128, dtype=torch.uint8, device="cuda")
        s["v"] = torch.full((pages, hk, d // 2, 4, 2, 8), 128, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.zeros(pages, hk, 2, device="cuda")
    s["k_tail"], s["v_tail"] = _randn(g, bt, hk, RING, d).half(), _randn(g, bt, hk, d, RING).half()
    if case["kind"] == "cache":
        s["q"] = (2 * _randn(g, bt, case["new"], case["heads"] * d)).half()
        s["o"] = torch.zeros_like(s["q"])
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / case["heads"]) for i in range(case["heads"])],
                                   device="cuda") if case["slopes"] else None
    else:
        kv = _randn(g, bt, case["new"], 2 * hk * d)
        s["kv"] = kv.half() if case["f16"] else kv
        first = [n // BLOCK * BLOCK for n in lens]
        s["first"], s["total"] = _ints(first), _ints([n + m for n, m in zip(lens, new)])
        s["span"] = max(n + m - f for n, m, f in zip(lens, new, first))
        s["out"] = [torch.zeros(bt, hk, s["span"], d, dtype=torch.float16, device="cuda") for _ in range(2)]
    return s


def _prepare_logits(case, seed):
    g, rows, vocab, hist = _gen(seed), case["rows"], case["vocab"], case["hist"]
    dt = torch.float16 if case["f16"] else torch.float32
    s = {"case": case, "x": (4 * _randn(g, rows, vocab)).to(dt)}
    if hist:
        # tokens repeat themselves: a few hundred ids make up most of a history
        near = torch.randint(0, vocab, (rows, 300), generator=g, device="cuda")
        pick = torch.randint(0, 300, (rows, hist), generator=g, device="cuda")
        far = torch.randint(0, vocab, (rows, hist), generator=g, device="cuda")
        rare = torch.rand(rows, hist, generator=g, device="cuda") < 0.2
        s["hist"] = torch.where(rare, far, near.gather(1, pick)).to(torch.int32)
        r = random.Random(seed)
        s["hist_len"] = _ints([hist] + [r.randint(0, hist) for _ in range(rows - 1)])
    s["rep"] = 1 + 0.5 * torch.rand(rows, generator=g, device="cuda")
    s["freq"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
    s["pres"] = torch.rand(rows, generator=g, device="cuda")
    if case["bias"] != "none":
        b = _randn(g, rows if case["bias"] == "row" else 1, vocab)
        s["bias"] = torch.where(torch.rand(b.shape, generator=g, device="cuda") < 0.05, 3 * b, torch.zeros_like(b))
    if case["mask"]:
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device="cuda").to(torch.int32)
    s["y"] = torch.zeros_like(s["x"])
    return s


def prepare(case, seed):
    s = {"attn": _prepare_attn, "append": _prepare_cache, "cache": _prepare_cache,
         "logits": _prepare_logits}[case["kind"]](case, seed)
    # device addresses, as a program that binds the C ABI holds them
    s["ptr"] = {k: v.data_ptr() for k, v in s.items() if torch.is_tensor(v)}
    return s


# ---- plain forms ----------------------------------------------------------------------------


def _views(s):
    """q [B,H,Sq,D], k and v [B,Hk,Sk,D] of an attention case, as they are stored"""
    case, at = s["case"], s["at"]
    bt, sq, sk, h, hk, d = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    q = s["rows"] if "rows" in s else s["q"]
    kv = s["rows"] if "rows" in s else s["kv"]
    part = lambda x, a, n, t: x[:, :, a:a + n * d].reshape(bt, t, n, d).transpose(1, 2)  # noqa: E731
    return part(q, at[0], h, sq), part(kv, at[1], hk, sk), part(kv, at[2], hk, sk)


def _softmax_v(sc, seen, v):
    """softmax over the seen keys, times v; rows that see none are 0"""
    sc = sc.masked_fill_(~seen, -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(p, v) / total, torch.zeros_like(total))


def _scores(q, k, case, slopes, pos, keys):
    """[B,Hk,G*Sq,Sk] -> [B,Hk,G,Sq,Sk] scores of grouped heads; pos: [Sq] or [B,1,1,Sq,1]"""
    bt, h, sq, d = q.shape
    hk = k.shape[1]
    sc = torch.matmul(q.reshape(bt, hk, h // hk * sq, d), k.transpose(-1, -2).contiguous())
    sc = sc.view(bt, hk, h // hk, sq, k.shape[2]).mul_(d ** -0.5)
    if case["cap"]:
        sc = sc.div_(case["cap"]).tanh_().mul_(case["cap"])
    if slopes is not None:
        sc = sc.sub_(slopes.view(1, hk, h // hk, 1, 1) * (pos - keys).abs())
    return sc


def _plain_attn(s):
    case = s["case"]
    bt, sq, sk, h, hk, d = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    q, k, v = (x.half().float() for x in _views(s))
    pos = torch.arange(sk - sq, sk, device="cuda")[:, None]
    keys = torch.arange(sk, device="cuda")[None, :]
    seen = torch.ones(1, sq, sk, dtype=torch.bool, device="cuda")
    if case["causal"]:
        seen = seen & (keys <= pos)
        if s["prefix"] is not None:
            seen = seen | (keys < s["prefix"].view(-1, 1, 1))
    if s["docs"] is not None:
        seen = seen & (s["docs"][:, sk - sq:, None] == s["docs"][:, None, :]) & (s["docs"][:, None, :] >= 0)
    sc = _scores(q, k, case, s["slopes"], pos, keys)
    o = _softmax_v(sc.view(bt, h, sq, sk), seen[:, None], v.repeat_interleave(h // hk, 1))
    return o.transpose(1, 2).reshape(bt, sq, h * d).to(s["o"].dtype)


def _dequantized(s, nb):
    """k, v [B,Hk,nb * 32,D] of the tables' first nb blocks"""
    case, pages = s["case"], s["table"][:, :nb].clamp(min=0).long()
    bt, hk, d = (case[k] for k in ("batch", "kv_heads", "dim"))
    out = []
    for codes, i in ((s["k"], 0), (_from_v_layout(s["v"], d), 1)):
        x = (codes[pages].float() - 128) * s["scales"][pages][..., i][..., None, None]
        out.append(x.transpose(1, 2).reshape(bt, hk, nb * BLOCK, d))
    return out


def _ring(s, pos):
    """k, v [B,Hk,n,D] of the fp16 ring at positions pos [B,n]"""
    bt, hk, d = (s["case"][k] for k in ("batch", "kv_heads", "dim"))
    slot = (pos % RING)[:, None, :, None].expand(bt, hk, pos.shape[1], d)
    return s["k_tail"].gather(2, slot), s["v_tail"].transpose(2, 3).gather(2, slot)


def _plain_append(s):
    case = s["case"]
    bt, hk, d, n = (case[k] for k in ("batch", "kv_heads", "dim", "new"))
    span = -(-s["span"] // BLOCK) * BLOCK
    pos = s["first"][:, None].long() + torch.arange(span, device="cuda")
    at = pos - s["lens"][:, None]                                   # index among the new tokens
    here = (pos < s["total"][:, None])[:, None, :, None]
    x = s["kv"].half().view(bt, n, 2, hk, d).permute(2, 0, 3, 1, 4)  # [2][B][Hk][n][D]
    pick = at.clamp(0, n - 1)[:, None, :, None].expand(bt, hk, span, d)
    whole = ((s["first"][:, None] + torch.arange(BLOCK, span + 1, BLOCK, device="cuda")) <= s["total"][:, None])
    out = []
    for kv, old, o in zip(x, _ring(s, pos), s["out"]):
        raw = torch.where((at < 0)[:, None, :, None], old, kv.gather(2, pick))
        y = torch.where(here, raw, torch.zeros_like(raw)).view(bt, hk, span // BLOCK, BLOCK, d)
        scale = (y.abs().amax((-1, -2)).double() / 127).float()[..., None, None]
        t = y.double() / scale                       # next to a border 32 bits would take the other code
        code = torch.sign(t) * torch.floor(t.abs() + 0.5)
        val = torch.where(scale > 0, code, torch.zeros_like(code)).float() * scale
        val = torch.where(whole[:, None, :, None, None], val, y.float()).view(bt, hk, span, d)
        o.copy_(torch.where(here, val, torch.zeros_like(val))[:, :, :s["span"]])
    return s["out"]


def _plain_cache(s):
    case = s["case"]
    bt, n, h, hk, d = (case[k] for k in ("batch", "new", "heads", "kv_heads", "dim"))
    total = (s["lens"] + s["new"])[:, None]
    keys = torch.arange(s["blocks"] * BLOCK, device="cuda")
    k, v = _dequantized(s, s["blocks"])
    rk, rv = _ring(s, keys[None].expand(bt, -1))
    raw = (keys[None] >= total // BLOCK * BLOCK)[:, None, :, None]
    k, v = torch.where(raw, rk.float(), k), torch.where(raw, rv.float(), v)
    live = (keys[None] < total)[:, None, :, None]
    k, v = k.masked_fill(~live, 0), v.masked_fill(~live, 0)
    pos = (s["lens"][:, None] + torch.arange(n, device="cuda"))[:, None, None, :, None]
    q = s["q"].float().view(bt, n, h, d).transpose(1, 2)
    sc = _scores(q, k, case, s["slopes"], pos, keys)
    seen = (keys <= pos).expand(bt, 1, h // hk, n, -1).reshape(bt, 1, h // hk * n, -1)
    o = _softmax_v(sc.view(bt, hk, h // hk * n, -1), seen, v).view(bt, h, n, d).transpose(1, 2).reshape(bt, n, h * d)
    mine = torch.arange(n, device="cuda")[None, :] < s["new"][:, None]  # a sequence's own rows; the others stay as they were
    return torch.where(mine[:, :, None], o.half(), torch.zeros_like(s["o"]))


def _plain_logits(s):
    case, x = s["case"], s["x"].float()
    rows, vocab, hist = case["rows"], case["vocab"], case["hist"]
    if hist:
        live = (torch.arange(hist, device="cuda") < s["hist_len"][:, None]).float()
        n = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, s["hist"].long(), live)
        x = torch.where(n > 0, torch.where(x > 0, x / s["rep"][:, None], x * s["rep"][:, None]), x)
        x = x - torch.where(n > 0, s["freq"][:, None] * n + s["pres"][:, None], torch.zeros_like(n))
    if "bias" in s:
        x = x + s["bias"]
    if "allowed" in s:
        v = torch.arange(vocab, device="cuda")
        x = x.masked_fill(((s["allowed"][:, v // 32] >> (v % 32)) & 1) == 0, -math.inf)
    return x.to(s["x"].dtype)


# ---- the framework's calls --------------------------------------------------------------------

_CTX = []


def _ctx():
    """the program's one kernel context"""
    if not _CTX:
        import edge_maskgit_amd as ema
        _CTX.append(ema.Context(0))
    return _CTX[0]


def _own_attn(s):
    case, p, at = s["case"], s["ptr"], s["at"]
    bt, sq, sk, h, hk, d = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    e = 2 if case["f16"] else 4
    q, kv = (p["rows"], p["rows"]) if "rows" in p else (p["q"], p["kv"])
    o = dict(o16=p["o"]) if case["f16"] else dict(o=p["o"])
    _ctx().attn_masked(q + e * at[0], kv + e * at[1], kv + e * at[2], s["q_st"], s["kv_st"], d, sq, sk, h, hk, bt, d ** -0.5,
                       in16=case["f16"], cap=case["cap"], slopes=p.get("slopes"), causal=case["causal"],
                       prefix=p.get("prefix"), docs=p.get("docs"), doc_stride=sk, o_strides=(1, h * d, d, sq * h * d), **o)
    return s["o"]


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
    hk, d, n = case["kv_heads"], case["dim"], case["new"]
    w, e = 2 * hk * d, 2 if case["f16"] else 4
    c.kv8_append(kv8, p["kv"], p["kv"] + e * hk * d, (1, w, d, n * w), n, p["lens"], p["new"], in16=case["f16"])
    c.kv8_read(kv8, p["first"], s["span"], p["total"], k16=s["out"][0].data_ptr(), v16=s["out"][1].data_ptr())
    return s["out"]


def _own_cache(s):
    case, p = s["case"], s["ptr"]
    n, h, d = case["new"], case["heads"], case["dim"]
    st = (1, h * d, d, n * h * d)
    _ctx().kv8_attn(_handle(s), p["q"], st, n, p["lens"], p["new"], h, d ** -0.5, in16=True, cap=case["cap"],
                    slopes=p.get("slopes"), o16=p["o"], o_strides=st)
    return s["o"]


def _own_logits(s):
    case, p = s["case"], s["ptr"]
    rows, vocab, hist = case["rows"], case["vocab"], case["hist"]
    _ctx().logits_process(p["x"], rows, vocab, p["y"], f16=case["f16"], hist=p.get("hist"), hist_len=p.get("hist_len"),
                          max_hist=hist, rep=p["rep"], freq=p["freq"], pres=p["pres"], bias=p.get("bias"),
                          bias_stride=vocab if case["bias"] == "row" else 0, allowed=p.get("allowed"),
                          allowed_stride=-(-vocab // 32))
    return s["y"]


def run(state):
    kind = state["case"]["kind"]
    if kind == "attn":
        return _own_attn(state) if own else _plain_attn(state)
    if kind == "append":
        return _own_append(state) if own else _plain_append(state)
    if kind == "cache":
        return _own_cache(state) if own else _plain_cache(state)
    return _own_logits(state) if own else _plain_logits(state)


# ---- what a pass cannot do without --------------------------------------------------------------


def _pairs(case):
    """visible (query, key) pairs of one head, all sequences"""
    sq, sk, off, n = case["sq"], case["sk"], case["sk"] - case["sq"], 0
    ids = _doc_ids(case) if case["docs"] else [[0] * sk] * case["batch"]
    for b, pre in enumerate(_prefixes(case)):
        spans, at = [], 0
        while at < sk:                                  # runs of one document
            end = at
            while end < sk and ids[b][end] == ids[b][at]:
                end += 1
            if ids[b][at] >= 0:
                spans.append((at, end))
            at = end
        for lo, hi in spans:
            for p in range(max(lo, off), hi):
                n += min(hi, max(p + 1, pre)) - lo if case["causal"] and max(p + 1, pre) > lo else 0 if case["causal"] else hi - lo
    return n


def work(case):
    if case["kind"] == "attn":
        bt, sq, sk, h, hk, d = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
        e = 2 if case["f16"] else 4
        return {"bytes": e * d * bt * (2 * h * sq + 2 * hk * sk), "flops": 4 * d * h * _pairs(case)}
    if case["kind"] == "append":
        # new tokens in, codes (or fp16) out; then the touched blocks' codes in, their values out
        hk, d, e = case["kv_heads"], case["dim"], 2 if case["f16"] else 4
        n, span = sum(_new(case)), sum(m + t % BLOCK for t, m in zip(_past(case), _new(case)))
        return {"bytes": 2 * hk * d * (n * e + span * (1 + 1 + 2)), "flops": 2 * hk * d * 4 * span}
    if case["kind"] == "cache":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        total = [t + m for t, m in zip(_past(case), _new(case))]
        by = sum(2 * hk * d * (t + t % BLOCK) + 8 * hk * (t // BLOCK) + 4 * -(-t // BLOCK) for t in total)
        return {"bytes": by + 4 * h * d * sum(_new(case)), "flops": sum(4 * d * h * t * m for t, m in zip(total, _new(case)))}
    rows, vocab = case["rows"], case["vocab"]
    e = 2 if case["f16"] else 4
    bias = {"none": 0, "shared": 1, "row": rows}[case["bias"]] * vocab * 4
    return {"bytes": 2 * rows * vocab * e + bias + (rows * -(-vocab // 32) * 4 if case["mask"] else 0) + 4 * rows * case["hist"],
            "flops": 4 * rows * vocab}


# ---- the definition in 64 bits ---------------------------------------------------------------


def _rows64(q, k, v, scale, cap, slope, dist, seen):
    """one head: q [n,D], k, v [t,D], dist and seen [n,t]"""
    s = (q @ k.t().contiguous()) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if slope is not None:
        s = s - slope * dist
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    m = s.max(-1, keepdim=True).values
    w = torch.where(seen, torch.exp(s - m), torch.zeros_like(s))
    z = w.sum(-1, keepdim=True)
    return torch.where(seen.any(-1, keepdim=True), (w @ v) / torch.where(z > 0, z, torch.ones_like(z)), torch.zeros_like(q))


def _exact_attn(case, s):
    bt, sq, sk, h, hk, d = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    q, k, v = _views(s)
    p, j = torch.arange(sq, device="cuda")[:, None] + sk - sq, torch.arange(sk, device="cuda")[None, :]
    out = torch.empty(bt, sq, h, d, dtype=torch.float64, device="cuda")
    for b in range(bt):
        seen = torch.ones(sq, sk, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = j <= torch.clamp(p, min=_prefixes(case)[b] - 1)
        if case["docs"]:
            ids = torch.tensor(_doc_ids(case)[b], device="cuda")
            seen = seen & (ids[p] == ids[j]) & (ids[j] != -1)
        for i in range(h):
            slope = 2.0 ** (-8.0 * (i + 1) / h) if case["slopes"] else None
            if slope is not None:
                slope = float(torch.tensor(slope, dtype=torch.float32))
            a = i // (h // hk)
            out[b, :, i] = _rows64(q[b, i].half().double(), k[b, a].half().double(), v[b, a].half().double(), d ** -0.5,
                                   case["cap"], slope, (p - j).abs(), seen)
    return out.reshape(bt, sq, h * d)


def _token_values(s, b, n, have):
    """k, v [Hk,n,D] in 64 bits of sequence b's first n tokens in a cache that holds `have`"""
    d, cut = s["case"]["dim"], have // BLOCK * BLOCK
    t = torch.arange(n, device="cuda")
    page = s["table"][b].long()[t // BLOCK].clamp(min=0)
    tok, ring = t % BLOCK, t % RING
    f = torch.arange(d, device="cuda")
    kc = s["k"][page, :, tok].double() - 128                                             # [n][Hk][D]
    vc = s["v"].view(s["pages"], -1, d * BLOCK)[page]                                     # [n][Hk][D * 32]
    at = ((f[None, :] // 2) * 4 + tok[:, None] // 8) * 16 + (f[None, :] % 2) * 8 + tok[:, None] % 8
    vc = vc.gather(2, at[:, None, :].expand(-1, vc.shape[1], -1)).double() - 128
    sc = s["scales"][page].double()                                                       # [n][Hk][2]
    old = (t < cut)[:, None, None]
    k = torch.where(old, kc * sc[..., :1], s["k_tail"][b][:, ring].transpose(0, 1).double())
    v = torch.where(old, vc * sc[..., 1:], s["v_tail"][b][:, :, ring].permute(2, 0, 1).double())
    return k.transpose(0, 1), v.transpose(0, 1)


def _exact_cache(case, s):
    n, h, hk, d = (case[k] for k in ("new", "heads", "kv_heads", "dim"))
    out = torch.zeros(case["batch"], n, h, d, dtype=torch.float64, device="cuda")
    for b, (past, m) in enumerate(zip(_past(case), _new(case))):
        k, v = _long_values(s, b, past + m)
        p, j = past + torch.arange(m, device="cuda")[:, None], torch.arange(past + m, device="cuda")[None, :]
        for i in range(h):
            slope = float(torch.tensor(2.0 ** (-8.0 * (i + 1) / h), dtype=torch.float32)) if case["slopes"] else None
            q = s["q"][b, :m, i * d:(i + 1) * d].double()
            a = i // (h // hk)
            out[b, :m, i] = _rows64(q, k[a], v[a], d ** -0.5, case["cap"], slope, (p - j).abs(), j <= p)
    return out.reshape(case["batch"], n, h * d)


def _long_values(s, b, n):
    """_token_values of a sequence, 4096 tokens at a time (each gathers the 32 tokens of its block)"""
    ks, vs = [], []
    whole = s["table"]
    for t0 in range(0, n, 4096):
        part = dict(s, table=whole[:, t0 // BLOCK:(t0 + 4096) // BLOCK])
        k, v = _token_values(part, b, min(4096, n - t0), max(0, n - t0))
        ks.append(k)
        vs.append(v)
    return torch.cat(ks, 1), torch.cat(vs, 1)


def _exact_append(case, s):
    hk, d = case["kv_heads"], case["dim"]
    outs = [torch.zeros(case["batch"], hk, s["span"], d, dtype=torch.float64, device="cuda") for _ in range(2)]
    for b, (past, m) in enumerate(zip(_past(case), _new(case))):
        lo = past // BLOCK * BLOCK
        slots = torch.arange(lo, past, device="cuda") % RING
        new = s["kv"][b, :m].half().double().view(m, 2, hk, d)
        for which in range(2):
            tail = s["k_tail"][b][:, slots] if which == 0 else s["v_tail"][b][:, :, slots].transpose(1, 2)
            x = torch.cat((tail.double(), new[:, which].transpose(0, 1)), 1)              # [Hk][tokens][D]
            for t in range(0, (past + m - lo) // BLOCK * BLOCK, BLOCK):
                blk = x[:, t:t + BLOCK]
                unit = (blk.abs().flatten(1).max(1).values / 127).float().double()[:, None, None]
                near = torch.trunc(blk / unit)
                near = near + torch.sign(blk) * ((blk / unit - near).abs() >= 0.5)
                x[:, t:t + BLOCK] = torch.where(unit > 0, near * unit, torch.zeros_like(blk))
            outs[which][b, :, :x.shape[1]] = x
    return outs


def _exact_logits(case, s):
    x = s["x"].double()
    if case["hist"]:
        for r in range(case["rows"]):
            n = torch.bincount(s["hist"][r, :int(s["hist_len"][r])].long(), minlength=case["vocab"]).double()
            rep, f, p = (float(s[k][r]) for k in ("rep", "freq", "pres"))
            y = torch.where(x[r] > 0, x[r] / rep, x[r] * rep) - f * n - p
            x[r] = torch.where(n > 0, y, x[r])
    if "bias" in s:
        x = x + s["bias"].double()
    if "allowed" in s:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device="cuda")) & 1
        x[bits.flatten(1)[:, :case["vocab"]] == 0] = -math.inf
    return x


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "append": _exact_append, "cache": _exact_cache, "logits": _exact_logits}[case["kind"]](case, s)
