"""Serving a decoder layer from a cache of 4-bit keys and values: the operators that stand between the q / k / v projections and
the output projection of a serving step, as cases to be timed and compared.

  rotary   norms of q and k per head and the rotation by position, in one pass (``qk_norm_rope``)
  cache    keys and values of new tokens quantised into cache pages (``kv4_append``) and read back as values (``kv4_read``)
  attend   attention of the newest tokens of every sequence over its pages (``kv4_attention``)
  pages    pages copied inside a cache, for forks and for compaction (``copy_pages``)

``listed()`` names twelve cases, ``draw(rng)`` makes another one of the same ranges. ``run`` computes a case in elementary torch
operations, or, where ``own`` is true, by the package's operators.

The cache. One uint8 tensor [pages, kv heads, page size / 16, 18 D]; the last dimension is a tile of 16 tokens of one head: D/2
bytes of key codes per token, then D/2 bytes of value codes per token, then per token and group of 64 channels the keys' fp16
(scale, least value) pairs, then the values'. A value is code * scale + least. In a token's key codes the 32-bit word w of chunk t
(four chunks) holds channels 32w + 8t + i, i = 0..7 from the low bits up; in its value codes the word w of chunk g (eight chunks)
holds channels 64w + 8g + i. The value codes of token r lie in row 4c + t, t = (r >> 1) & 3, c = (r & 1) + 2 (r >> 3), and their
chunk g at place g ^ 2t. Token i of a sequence is token i % page size of page page_table[sequence, i / page size].
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
LARGEST = 65504.0  # of fp16: what the cache's scales can stand for
TABLE = 65536  # positions of the rotation tables


def listed():
    return [
        # A decoding step of a small batch: one token per sequence, bound by latency.
        {"name": "rotary 16x32+8x128 bf16", "kind": "rotary", "tokens": 16, "hq": 32, "hk": 8, "d": 128, "rot": 128, "axes": 1, "dtype": "bf16"},
        # A prompt batch of the size of the package's decoder layer, positions of images and video (time, height, width).
        {"name": "rotary 16384x32+8x128 bf16 3 axes", "kind": "rotary", "tokens": 16384, "hq": 32, "hk": 8, "d": 128, "rot": 128, "axes": 3, "dtype": "bf16"},
        # The encoder block's heads in fp32, half of every head rotated, a number of tokens that is no multiple of anything.
        {"name": "rotary 1237x4+4x64 f32 half", "kind": "rotary", "tokens": 1237, "hq": 4, "hk": 4, "d": 64, "rot": 32, "axes": 1, "dtype": "f32"},
        # One new token for each of 64 sequences: every one goes to another page.
        {"name": "cache 64x8x128 bf16", "kind": "cache", "tokens": 64, "hk": 8, "d": 128, "page": 64, "dtype": "bf16", "spread": True},
        # The prompts of a prefill batch.
        {"name": "cache 16384x8x128 bf16", "kind": "cache", "tokens": 16384, "hk": 8, "d": 128, "page": 64, "dtype": "bf16", "spread": False},
        # A request that is alone: one token, a short history, every head with keys of its own.
        {"name": "attend 1x1 of 333 32/32x128 bf16", "kind": "attend", "batch": 1, "new": 1, "longest": 333, "shortest": 333, "hk": 32, "group": 1, "d": 128,
         "page": 16, "dtype": "bf16"},
        # A decoding step of a serving batch with histories of all lengths.
        {"name": "attend 64x1 of 8192 32/8x128 bf16", "kind": "attend", "batch": 64, "new": 1, "longest": 8192, "shortest": 512, "hk": 8, "group": 4, "d": 128,
         "page": 64, "dtype": "bf16"},
        # A few very long histories: the cache read once is all there is.
        {"name": "attend 4x1 of 131072 32/8x128 f16", "kind": "attend", "batch": 4, "new": 1, "longest": 131072, "shortest": 100001, "hk": 8, "group": 4, "d": 128,
         "page": 128, "dtype": "f16"},
        # Drafted tokens checked together: a few new tokens per sequence, small heads.
        {"name": "attend 24x5 of 3001 16/4x64 f16", "kind": "attend", "batch": 24, "new": 5, "longest": 3001, "shortest": 7, "hk": 4, "group": 4, "d": 64,
         "page": 32, "dtype": "f16"},
        # Chunks of long prompts: up to 2048 new tokens behind what is in the cache already.
        {"name": "attend 3x2048 of 8192 32/8x128 bf16", "kind": "attend", "batch": 3, "new": 2048, "longest": 8192, "shortest": 2500, "hk": 8, "group": 4, "d": 128,
         "page": 64, "dtype": "bf16"},
        # A sequence is forked: the pages that both sides go on writing to are copied.
        {"name": "pages 6 of 8x64x128", "kind": "pages", "count": 6, "pages": 512, "hk": 8, "d": 128, "page": 64},
        # Compaction after many requests have ended.
        {"name": "pages 1500 of 8x64x128", "kind": "pages", "count": 1500, "pages": 4096, "hk": 8, "d": 128, "page": 64},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotary", "cache", "attend", "attend", "attend", "pages"])
    d = rng.choice([64, 128, 128, 256])
    if kind == "rotary":
        hk = rng.choice([1, 2, 4, 8])
        hq, d = hk * rng.choice([1, 2, 4]), rng.choice([64, 80, 96, 128, 128, 256])
        most = 16384 * 40 * 128 // ((hq + hk) * d)
        return {"kind": kind, "tokens": _log_int(rng, 1, min(32768, most)), "hq": hq, "hk": hk, "d": d, "rot": rng.choice([d, d, d // 2]),
                "axes": rng.choice([1, 1, 3]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if kind == "cache":
        hk = rng.choice([1, 2, 4, 8])
        return {"kind": kind, "tokens": _log_int(rng, 1, 16384 * 8 * 128 // (hk * d)), "hk": hk, "d": d, "page": rng.choice([16, 32, 64, 128]),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "spread": rng.random() < 0.5}
    if kind == "pages":
        pages = _log_int(rng, 16, 4096)
        return {"kind": kind, "count": _log_int(rng, 1, max(1, pages * 3 // 8)), "pages": pages, "hk": rng.choice([1, 2, 4, 8]),
                "d": rng.choice([64, 128]), "page": rng.choice([16, 32, 64])}
    hk, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 5, 8])
    new = rng.choice([1, 1, 1, _log_int(rng, 2, 8), _log_int(rng, 16, 2048)])
    batch = _log_int(rng, 1, 64 if new == 1 else 16)
    longest = _log_int(rng, 16, min(131072, 3 * 131072 * 8 * 128 // (batch * hk * d)))
    if new > 8:  # a chunk, at most the largest listed one's products
        longest = min(16384, max(longest, new))
        most = 2048 * 12000 * 32 * 128 // (longest * hk * group * d)
        batch = max(1, min(batch, most // new))
        new = min(new, most // batch)
    return {"kind": kind, "batch": batch, "new": new, "longest": longest, "shortest": max(1, longest // rng.choice([1, 4, 16])), "hk": hk, "group": group,
            "d": d, "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "bf16", "f16"])}


# ---- inputs ------------------------------------------------------------------------------------
def _generator(seed, device="cuda"):
    return torch.Generator(device).manual_seed(seed)


def _tables(rot):
    """cos and sin of every position and rotated channel [TABLE, rot], the two halves alike."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(TABLE, dtype=torch.float64, device="cuda")[:, None] * inv
    angle = torch.cat((angle, angle), 1)
    return angle.cos().float(), angle.sin().float()


def _sections(case):
    """Frequency pairs per axis: a quarter of them follow the time, the others height and width."""
    if case["axes"] == 1:
        return []
    pairs = case["rot"] // 2
    h = (pairs - pairs // 4) // 2
    return [pairs - 2 * h, h, h]


def _positions(case, g):
    n = case["tokens"]
    if case["axes"] == 1:
        return torch.randint(0, TABLE - n, (1,), generator=g, device="cuda") + torch.arange(n, device="cuda")
    frame = torch.arange(n, device="cuda")  # frames of 24 x 32 patches
    start = torch.randint(0, 1000, (1,), generator=g, device="cuda")
    return torch.stack((start + frame // 768, start + frame % 768 // 32, start + frame % 32))


def _keys_and_values(shape, g, dtype=torch.float32):
    """Keys with a few channels that stand out, as trained projections have them, and values."""
    k = torch.randn(shape, generator=g, device="cuda")
    v = torch.randn(shape, generator=g, device="cuda") * 0.5
    k[..., ::37] *= 4.0
    return k.to(dtype), v.to(dtype)


def _pages_of_values(pages, hk, tiles, d, g):
    """A cache [pages, hk, tiles, 18 d] that holds keys and values of the kind above, made 256 pages at a time."""
    cache = torch.empty(pages, hk, tiles, 18 * d, dtype=torch.uint8, device="cuda")
    for at in range(0, pages, 256):
        n = min(256, pages - at)
        k, v = _keys_and_values((n, hk, tiles, 16, d), g)
        cache[at:at + n] = _packed(k, v)
    return cache


def _value_places(d, device):
    """Where a token's 8-channel words of value codes lie: (rows [16], places [16, d / 8]) inside a tile."""
    r = torch.arange(16, device=device)
    t = (r >> 1) & 3
    row = 4 * ((r & 1) + 2 * (r >> 3)) + t
    j = torch.arange(d // 8, device=device)
    return row, ((j % 8)[None] ^ (2 * t)[:, None]) * (d // 64) + (j // 8)[None]


def _key_places(d, device):
    j = torch.arange(d // 8, device=device)
    return (j % 4) * (d // 32) + j // 4


def _packed(k, v):
    """Tiles [..., 18 d] of keys and values [..., 16, d]."""
    d, lead = k.shape[-1], k.shape[:-2]
    out = torch.empty(*lead, 18 * d, dtype=torch.uint8, device=k.device)
    row, place = _value_places(d, k.device)
    for i, x in enumerate((k, v)):
        code, scale, least = _quantised(x)
        word = code.to(torch.uint8).reshape(*lead, 16, d // 8, 4, 2)
        word = word[..., 0] | (word[..., 1] << 4)
        at = torch.empty_like(word)
        if i == 0:
            at[..., _key_places(d, k.device), :] = word
        else:
            at[..., row[:, None], place, :] = word
        out[..., 8 * d * i:8 * d * (i + 1)] = at.flatten(-3)
        pairs = torch.stack((scale, least), -1).contiguous().view(torch.uint8)
        out[..., (16 + i) * d:(17 + i) * d] = pairs.flatten(-3)
    return out


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "pages":
        cache = torch.randint(0, 256, (case["pages"], case["hk"], case["page"] // 16, 18 * case["d"]), generator=g, device="cuda", dtype=torch.uint8)
        pick = torch.randperm(case["pages"], generator=g, device="cuda")[:2 * case["count"]].tolist()
        return {"case": case, "cache": cache, "src": pick[:case["count"]], "dst": pick[case["count"]:]}
    dtype, d = DTYPES[case["dtype"]], case["d"]
    if kind == "rotary":
        hq, hk = case["hq"], case["hk"]
        qkv = torch.randn(case["tokens"], hq + 2 * hk, d, generator=g, device="cuda").to(dtype)  # the output of one packed projection
        cos, sin = _tables(case["rot"])
        weights = [(1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype) for _ in range(2)]
        return {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + hk], "wq": weights[0], "wk": weights[1], "cos": cos, "sin": sin,
                "positions": _positions(case, g), "sections": _sections(case)}
    hk, tiles = case["hk"], case["page"] // 16
    if kind == "cache":
        n, page = case["tokens"], case["page"]
        k, v = _keys_and_values((n, hk, d), g, dtype)
        pages = n + 8 if case["spread"] else -(-n // page) + 8
        order = torch.randperm(pages, generator=g, device="cuda")
        i = torch.arange(n, device="cuda")
        slots = order[i] * page + torch.randint(0, page, (n,), generator=g, device="cuda") if case["spread"] else order[i // page] * page + i % page
        return {"case": case, "k": k, "v": v, "slots": slots, "cache": torch.zeros(pages, hk, tiles, 18 * d, dtype=torch.uint8, device="cuda")}
    lens, new, at = _lengths(case, seed), [], [0]
    for n in lens:
        new.append(min(case["new"], n))
        at.append(at[-1] + new[-1])
    most = -(-max(lens) // case["page"])
    pages = sum(-(-n // case["page"]) for n in lens) + 8
    cache = _pages_of_values(pages, hk, tiles, d, g)
    order, table, used = torch.randperm(pages, generator=g, device="cuda"), torch.zeros(len(lens), most, dtype=torch.int64, device="cuda"), 0
    for b, n in enumerate(lens):
        count = -(-n // case["page"])
        table[b, :count] = order[used:used + count]
        used += count
    q = torch.randn(at[-1], hk * case["group"], d, generator=g, device="cuda").to(dtype)
    return {"case": case, "q": q, "cache": cache, "table": table, "lens": torch.tensor(lens, device="cuda"), "starts": torch.tensor(at, device="cuda"),
            "most_new": max(new), "most": max(lens)}


def _lengths(case, seed):
    """Histories between the case's shortest and longest, both of them there, the others evenly spread between."""
    r = torch.rand(case["batch"], generator=_generator(seed, "cpu"))
    lens = (case["shortest"] + r * (case["longest"] - case["shortest"])).round().int().tolist()
    lens[0] = case["longest"]
    if case["batch"] > 1:
        lens[-1] = case["shortest"]
    return lens


# ---- plain forms ---------------------------------------------------------------------------------
def _plain_rotary(s):
    case, cos, sin, pos = s["case"], s["cos"], s["sin"], s["positions"]
    half = case["rot"] // 2
    if s["sections"]:
        axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=pos.device), torch.tensor(s["sections"], device=pos.device))
        at = pos[axis].T  # [tokens, pairs]
        pair = torch.arange(half, device=pos.device)[None]
        c = torch.cat((cos[at, pair], cos[at, pair + half]), 1)[:, None]
        n = torch.cat((sin[at, pair], sin[at, pair + half]), 1)[:, None]
    else:
        c, n = cos[pos][:, None], sin[pos][:, None]

    def one(x, w):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
        r = y[..., :2 * half]
        turned = torch.cat((-r[..., half:], r[..., :half]), -1)
        return torch.cat((r * c + turned * n, y[..., 2 * half:]), -1).to(x.dtype)

    return one(s["q"], s["wq"]), one(s["k"], s["wk"])


def _quantised(x):
    """Codes (as floats), scales and least values (fp16) of [..., d], in groups of 64 channels."""
    y = x.float().clamp(-LARGEST, LARGEST).unflatten(-1, (-1, 64))
    least = y.amin(-1).half()
    scale = ((y.amax(-1) - least.float()) / 15.0).half()
    code = ((y - least.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 15)
    return torch.where(scale[..., None] > 0, code, 0.0).flatten(-2), scale, least


def _plain_cache(s):
    def one(x):
        code, scale, least = _quantised(x)
        return (code.unflatten(-1, (-1, 64)) * scale.float()[..., None] + least.float()[..., None]).flatten(-2).to(x.dtype)

    return one(s["k"]), one(s["v"])


def _unpacked(tiles):
    """Keys and values [..., 16, d] (fp32) of tiles [..., 18 d]."""
    d, lead = tiles.shape[-1] // 18, tiles.shape[:-1]
    row, place = _value_places(d, tiles.device)
    word = tiles[..., :16 * d].unflatten(-1, (2, 16, d // 8, 4))
    word = torch.stack((word & 15, word >> 4), -1).flatten(-2)
    pairs = tiles[..., 16 * d:].contiguous().view(torch.float16).unflatten(-1, (2, 16, d // 64, 2)).float()

    def one(i, codes):
        return (codes.flatten(-2).unflatten(-1, (-1, 64)).float() * pairs[..., i, :, :, :1] + pairs[..., i, :, :, 1:]).flatten(-2)

    return one(0, word[..., 0, :, :, :][..., _key_places(d, tiles.device), :]), one(1, word[..., 1, :, :, :][..., row[:, None], place, :])


def _plain_attend(s):
    case, q, lens, starts = s["case"], s["q"], s["lens"], s["starts"]
    hk, d = case["hk"], case["d"]
    batch, most_new, most = len(lens), s["most_new"], s["most"]
    k, v = _unpacked(s["cache"][s["table"]])  # [batch, pages, hk, tiles, 16, d]
    k, v = (x.transpose(1, 2).reshape(batch, hk, -1, d)[:, :, :most] for x in (k, v))
    new = starts[1:] - starts[:-1]
    i = torch.arange(most_new, device=q.device)
    there = i < new[:, None]
    rows = torch.where(there, starts[:-1, None] + i, 0)
    padded = q.float()[rows].reshape(batch, most_new, hk, -1, d).permute(0, 2, 3, 1, 4)  # [batch, hk, group, new, d]
    score = (padded.flatten(2, 3) @ k.transpose(-1, -2)).mul_(d ** -0.5).unflatten(2, (-1, most_new))
    visible = (lens - new)[:, None] + i + 1  # keys that a new token sees
    hidden = torch.arange(most, device=q.device) >= visible[:, :, None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    p = torch.div(p, p.sum(-1, keepdim=True), out=p)
    v = torch.where((torch.arange(most, device=q.device) < lens[:, None])[:, None, :, None], v, 0.0)
    out = (p.flatten(2, 3) @ v).unflatten(2, (-1, most_new)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[there].to(q.dtype)


def _plain_pages(s):
    at = torch.tensor([s["src"], s["dst"]], device="cuda")
    s["cache"][at[1]] = s["cache"][at[0]]
    return s["cache"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        from xpu_graph_b200 import ops

        if kind == "rotary":
            return ops.qk_norm_rope(state["q"], state["k"], state["wq"], state["wk"], EPS, state["cos"], state["sin"], state["positions"], state["sections"])
        if kind == "cache":
            ops.kv4_append(state["cache"], state["k"], state["v"], state["slots"])
            return ops.kv4_read(state["cache"], state["slots"], state["k"].dtype)
        if kind == "attend":
            return ops.kv4_attention(state["q"], state["cache"], state["table"], state["lens"], state["starts"], state["most_new"], state["case"]["d"] ** -0.5)
        ops.copy_pages(state["cache"], state["src"], state["dst"])
        return state["cache"]
    return {"rotary": _plain_rotary, "cache": _plain_cache, "attend": _plain_attend, "pages": _plain_pages}[kind](state)


def work(case):
    kind = case["kind"]
    if kind == "pages":
        return {"bytes": 2.0 * case["count"] * case["hk"] * case["page"] // 16 * 18 * case["d"], "flops": 0.0}
    size, d = SIZE[case["dtype"]], case["d"]
    if kind == "rotary":
        elements = case["tokens"] * (case["hq"] + case["hk"]) * d
        rows = case["tokens"] if case["axes"] == 1 else min(case["tokens"], case["tokens"] // 768 + 57)  # of the tables
        return {"bytes": 2.0 * elements * size + 8.0 * case["tokens"] * case["axes"] + 8.0 * rows * case["rot"], "flops": 10.0 * elements}
    if kind == "cache":  # values in, the cache written and read, values out
        elements = 2.0 * case["tokens"] * case["hk"] * d
        return {"bytes": 2.0 * elements * size + 2.0 * elements * 9 / 16 + 16.0 * case["tokens"], "flops": 8.0 * elements}
    lens = _lengths(case, 0)
    new = [min(case["new"], n) for n in lens]
    heads = case["hk"] * case["group"]
    pairs = sum(m * n - m * (m - 1) // 2 for m, n in zip(new, lens))
    return {"bytes": sum(lens) * case["hk"] * d * 9 / 8 + 2.0 * sum(new) * heads * d * size, "flops": 4.0 * pairs * heads * d}


# ---- the definitions in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "pages":  # whole numbers
        return None
    if kind == "rotary":
        out = []
        for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
            y = x.double()
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
            half, first = case["rot"] // 2, 0
            z = y.clone()
            for a, count in enumerate(s["sections"] or [half]):  # an axis turns its own pairs
                p = s["positions"][a] if s["sections"] else s["positions"]
                for lo, hi, sign in ((first, half + first, -1.0), (half + first, first, 1.0)):
                    c, n = (t[p][:, None, lo:lo + count].double() for t in (s["cos"], s["sin"]))
                    z[..., lo:lo + count] = y[..., lo:lo + count] * c + sign * y[..., hi:hi + count] * n
                first += count
            out.append(z)
        return out
    if kind == "cache":
        out = []
        for x in (s["k"], s["v"]):
            y = x.double().clamp(-LARGEST, LARGEST).reshape(-1, 64)
            least = y.min(1, keepdim=True).values.half().double()
            scale = ((y.max(1, keepdim=True).values - least) / 15).half().double()
            code = torch.clamp(torch.round((y - least) / torch.where(scale > 0, scale, 1.0)), 0, 15)
            out.append((torch.where(scale > 0, code, 0.0) * scale + least).reshape(x.shape))
        return out
    out, d, hk, group = [], case["d"], case["hk"], case["group"]
    for b, n in enumerate(s["lens"].tolist()):
        lo, hi = s["starts"][b].item(), s["starts"][b + 1].item()
        tiles = s["cache"][s["table"][b, :-(-n // case["page"])]].transpose(0, 1).reshape(hk, -1, 18 * d)
        k, v = _exact_values(tiles, d)
        q = s["q"][lo:hi].double().reshape(hi - lo, hk, group, d)
        last = torch.arange(n - (hi - lo), n, device="cuda")
        beyond = torch.arange(n, device="cuda")[None] > last[:, None]
        heads = []
        for h in range(hk):
            score = torch.einsum("igd,jd->gij", q[:, h], k[h, :n]) / math.sqrt(d)
            p = torch.softmax(score.masked_fill_(beyond, -math.inf), -1)
            heads.append(torch.einsum("gij,jd->igd", p, v[h, :n]))
        out.append(torch.stack(heads, 1).reshape(hi - lo, hk * group, d))
    return torch.cat(out)


def _exact_values(tiles, d):
    """Keys and values [hk, tokens, d] of tiles [hk, n, 18 d], channel by channel as the layout is written down."""
    c = torch.arange(d, device="cuda")
    r = torch.arange(16, device="cuda")[:, None]
    t = r // 2 % 4
    key = r * (d // 2) + 4 * (c // 8 % 4 * (d // 32) + c // 32) + c % 8 // 2
    value = 8 * d + (4 * (r % 2 + 2 * (r // 8)) + t) * (d // 2) + 4 * (torch.bitwise_xor(c // 8 % 8, 2 * t) * (d // 64) + c // 64) + c % 8 // 2
    out = []
    for i, at in enumerate((key, value)):
        code = (tiles[..., at.reshape(-1)].reshape(*tiles.shape[:-1], 16, d) >> (4 * (c % 2)).to(torch.uint8)) & 15
        pair = (tiles[..., (16 + i) * d:(17 + i) * d].contiguous().view(torch.float16).double()).reshape(*tiles.shape[:-1], 16, d // 64, 2)
        out.append((code.double() * pair[..., 0].repeat_interleave(64, -1) + pair[..., 1].repeat_interleave(64, -1)).flatten(-3, -2))
    return out
