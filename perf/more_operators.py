"""What further operators over a paged key-value cache are measured on: appending rotated rows, a cache held in 4 bits, attention over
the blocks that a cheap score selects.

The cache is two arrays [block][layer][key-value head][position in the block][head size] of f32 or f16, or in 4 bits ("q4_0"): 32
elements share an f16 scale d and have a code of 4 bits each, an element is (code - 8) d. The codes lie as above, half a byte an element,
eight to a little-endian word (element 2 i of the eight at bit 4 i, element 2 i + 1 at bit 16 + 4 i); the scales lie behind all codes as
[block][layer][key-value head][head size / 32][position in the block]. A sequence's position t lies in block table[t // kv_block].
`lens` counts a sequence's cached positions, the new ones among them: new row i of n stands at position len - n + i.

  append   q and k of new tokens turned by their positions' angles (a table of cosines and sines), q to rows, k and v into the cache,
           rounded to its type; from a 4-bit cache the new rows are read back, as a program hands a prefix on
  attend   softmax(scale q K^T) V for every new token over a 4-bit cache: token p sees t <= p, with a window only the last `window`
           positions and the first `sinks`
  bounds   of every block that holds new tokens, per layer and key-value head: the least and the largest value of each key element
  select   for every new token and key-value head: blocks get the largest score that their bounds allow a query head; the first `first`,
           the last `recent` and of the others the best are kept, `select` in all (ties to the lower), and attended to as above

Queries, keys and values are N(0, 1) as projections after a norm are; for `select` the keys of a block lie about a centre of its own, as
the keys of a passage do.
"""
import importlib
import math

import torch

own = False

# Most bytes and operations of a drawn pass, and bytes of what its plain form holds at a time: below the largest listed case's.
MOST_BYTES, MOST_FLOPS, MOST_HELD = 1.0e8, 2.0e11, 6.0e9


def listed():
    return [
        # chat with one user: a token's rows into an f32 cache, where only the call counts
        {"name": "append_1_token", "op": "append", "type": "f32", "heads": 32, "heads_kv": 8, "dim": 128, "rot": 128, "halves": False,
         "block": 16, "layers": 2, "seqs": 1, "new": 1, "len": 130, "offset": 0},
        # a server's step behind evictions: positions run ahead of places, part of a head is turned, halves paired, head size 80
        {"name": "append_32_ragged", "op": "append", "type": "f16", "heads": 24, "heads_kv": 4, "dim": 80, "rot": 64, "halves": True,
         "block": 20, "layers": 2, "seqs": 32, "new": 3, "len": 2000, "offset": 90000},
        # a prompt chunk of the device session's largest size into a 4-bit cache, read back
        {"name": "append_512_q4", "op": "append", "type": "q4_0", "heads": 32, "heads_kv": 8, "dim": 128, "rot": 128, "halves": False,
         "block": 16, "layers": 2, "seqs": 1, "new": 512, "len": 900, "offset": 0},
        # chat with one user, a short history: the smallest attention
        {"name": "decode_1_short", "op": "attend", "type": "q4_0", "heads": 32, "heads_kv": 8, "dim": 128, "block": 16, "layers": 2,
         "seqs": 1, "new": 1, "len": 200, "window": 0, "sinks": 0},
        # one user, a whole book in the cache
        {"name": "decode_1_long", "op": "attend", "type": "q4_0", "heads": 32, "heads_kv": 8, "dim": 128, "block": 64, "layers": 1,
         "seqs": 1, "new": 1, "len": 100003, "window": 0, "sinks": 0},
        # a server's step with a half-billion-parameter model: sequences of every length, seven query heads a key, blocks of no power of two
        {"name": "decode_32_ragged", "op": "attend", "type": "q4_0", "heads": 14, "heads_kv": 2, "dim": 64, "block": 20, "layers": 2,
         "seqs": 32, "new": 1, "len": 8192, "window": 0, "sinks": 0},
        # a long document's next chunk: bound by the matrix cores
        {"name": "chunk_2048", "op": "attend", "type": "q4_0", "heads": 32, "heads_kv": 8, "dim": 128, "block": 64, "layers": 1,
         "seqs": 1, "new": 2048, "len": 8192, "window": 0, "sinks": 0},
        # several prompts at once, none a whole tile, a window inside them
        {"name": "chunk_ragged_window", "op": "attend", "type": "q4_0", "heads": 12, "heads_kv": 4, "dim": 96, "block": 24, "layers": 2,
         "seqs": 5, "new": 401, "len": 1201, "window": 300, "sinks": 4},
        # a server's step: one block a sequence
        {"name": "bounds_step", "op": "bounds", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 32, "layers": 2,
         "seqs": 32, "new": 1, "len": 4000},
        # a long prompt's blocks in an f32 cache
        {"name": "bounds_prompt", "op": "bounds", "type": "f32", "heads": 32, "heads_kv": 8, "dim": 128, "block": 64, "layers": 1,
         "seqs": 1, "new": 8000, "len": 8190},
        # one user behind a whole book: 32 of 1563 blocks
        {"name": "select_1_long", "op": "select", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 64, "layers": 1,
         "seqs": 1, "new": 1, "len": 100003, "select": 32, "first": 1, "recent": 2},
        # a server's step over 4-bit caches, a few tokens a sequence as when drafts are checked, blocks of twenty
        {"name": "select_8_ragged", "op": "select", "type": "q4_0", "heads": 16, "heads_kv": 4, "dim": 64, "block": 20, "layers": 2,
         "seqs": 8, "new": 5, "len": 16000, "select": 48, "first": 1, "recent": 2},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "bounds", "select", "select"])
    kind = "q4_0" if op == "attend" else rng.choice(["f32", "f16", "q4_0"])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 256] if kind == "q4_0" else [40, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    c = {"op": op, "type": kind, "heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "heads_kv": kv, "dim": dim,
         "block": rng.choice([8, 16, 16, 20, 32, 64, 128]) if op in ("bounds", "select") else rng.choice([1, 16, 16, 20, 32, 64, 128]),
         "layers": rng.choice([1, 2, 3]), "seqs": _log(rng, 1, 16 if op == "select" else 64)}
    c["new"] = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 2, 48) if op == "select" else _log(rng, 16, 1024)])
    c["len"] = c["new"] + _log(rng, 1, 65536 if c["seqs"] <= 4 and c["new"] < 16 else 8192)
    if op == "select":
        c["len"] = c["new"] + _log(rng, 300, 131072 if c["seqs"] <= 4 else 16384)
    if op == "append":
        c.update(rot=rng.choice([dim, dim, 2 * (dim // 4)]), halves=rng.random() < 0.5, offset=rng.choice([0, 0, _log(rng, 1, 131072)]))
    if op == "attend":
        c["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
        c["sinks"] = rng.choice([0, 4]) if c["window"] else 0
    if op == "select":
        c.update(first=rng.choice([0, 1]), recent=rng.choice([1, 2, 4]))
        c["select"] = c["first"] + c["recent"] + max(1, _log(rng, 64, 2048) // c["block"])
    # fewer, then shorter sequences until the pass fits
    while _cost(c) > 1.0:
        if c["seqs"] > 1:
            c["seqs"] = (c["seqs"] + 1) // 2
        else:
            c["new"] = (c["new"] + 1) // 2
            c["len"] = max(c["new"] + 1, c["len"] // 2)
    return c


def _cost(c):
    w = work(c)
    held = _slots(c) * c["layers"] * c["heads_kv"] * c["dim"] * 8.0
    if c["op"] == "attend":
        held = max(held, 8.0 * c["seqs"] * c["new"] * c["heads"] * c["len"])
    if c["op"] == "select":
        held = max(held, c["seqs"] * c["new"] * c["heads_kv"] * (16.0 * c["select"] * c["block"] * c["dim"] + 16.0 * c["heads"] * c["len"] / c["block"]))
    return max(w["bytes"] / MOST_BYTES, w["flops"] / MOST_FLOPS, held / MOST_HELD)


# ------------------------------------------------------------------ shapes: the lengths follow from the case, their order from the seed
def _lens(c):
    """Cached positions of every sequence, spread evenly up to the longest."""
    n, least = c["seqs"], c["new"]
    return [least + (c["len"] - least) * (b + 1) // n for b in range(n)]


def _news(c):
    """New tokens of every sequence: as many for each, except that the chunks of several prompts differ."""
    n, most = c["seqs"], c["new"]
    return [most] * n if most <= 1 else [max(1, most * (b + 1) // n) for b in range(n)]


def _slots(c):
    return (sum(-(-x // c["block"]) for x in _lens(c)) + 3) * c["block"]


def _size(c):
    """Bytes of an element of the cache."""
    return {"f32": 4, "f16": 2, "q4_0": 18 / 32}[c["type"]]


def _visible(c):
    """Pairs of a token and a position it sees, and positions that any token of the call sees."""
    pairs = seen = 0
    w, k = c["window"], c["sinks"]
    for length, new in zip(_lens(c), _news(c)):
        for p in range(length - new, length):
            pairs += p + 1 if not w else min(p + 1, w) + min(k, max(0, p + 1 - w))
        seen += length if not w else length - max(0, (length - new + 1 - w) - min(k, max(0, length - new + 1 - w)))
    return pairs, seen


def work(case):
    c = case
    kv, d, tokens = c["heads_kv"], c["dim"], sum(_news(c))
    tables = 4 * sum(-(-x // c["block"]) for x in _lens(c))
    if c["op"] == "append":
        rows = tokens * kv * d
        back = rows * (2 * _size(c) + 8) if c["type"] == "q4_0" else 0
        return {"bytes": int(8 * tokens * c["heads"] * d + rows * (8 + 2 * _size(c)) + back + 4 * tokens * c["rot"]) + tables,
                "flops": 3 * tokens * (c["heads"] + kv) * c["rot"]}
    bound = 2 * d * (4 if c["type"] == "f32" else 2)  # bytes of a block's bounds
    if c["op"] == "bounds":
        read = wrote = 0
        for length, new in zip(_lens(c), _news(c)):
            from_block, to_block = (length - new) // c["block"], (length - 1) // c["block"] + 1
            read += length - from_block * c["block"]
            wrote += to_block - from_block
        return {"bytes": int(kv * (read * d * _size(c) + wrote * bound)) + tables, "flops": 2 * kv * read * d}
    if c["op"] == "select":
        total, flops = 0.0, 0
        for length, new in zip(_lens(c), _news(c)):
            blocks, kept = -(-length // c["block"]), min(length, c["select"] * c["block"])
            scored = max(0, blocks - c["first"] - c["recent"]) if blocks > c["select"] else 0
            total += kv * (scored * bound + 2 * kept * d * _size(c))  # what one token reads: others' blocks may be the same ones
            flops += new * c["heads"] * d * (2 * scored + 4 * kept)
        return {"bytes": int(total + 8 * tokens * c["heads"] * d + 4 * tokens * kv * c["select"]) + tables, "flops": flops}
    pairs, seen = _visible(c)
    return {"bytes": int(2 * seen * kv * d * _size(c) + 8 * tokens * c["heads"] * d) + tables, "flops": 4 * pairs * c["heads"] * d}


# ------------------------------------------------------------------ four bits
def _pack(x):
    """Codes [..., d / 2] (bytes) and scales [..., d / 32] of x [..., d]: d = minus an eighth of the element of largest size (the first of
    them), to 8 significant bits, so that every multiple up to eight is an f16; codes are the nearest, ties to even."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    size = b.abs()
    at = torch.where(size == size.amax(-1, keepdim=True), torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    scale = (b.gather(-1, at) / -8).bfloat16().float().clamp(-8160, 8160).half()
    d = scale.double()
    c = torch.where(d != 0, torch.round(b.double() / torch.where(d != 0, d, torch.ones_like(d))), torch.zeros_like(b, dtype=torch.float64))
    c = (c + 8).clamp(0, 15).to(torch.int32).reshape(*b.shape[:-1], 4, 4, 2)
    shift = torch.tensor([[4 * i, 16 + 4 * i] for i in range(4)], dtype=torch.int32, device=x.device)
    words = (c << shift).sum((-1, -2), dtype=torch.int64).to(torch.int32)  # [..., blocks, 4]
    return words.reshape(*x.shape[:-1], -1).contiguous().view(torch.uint8), scale.squeeze(-1)


def _unpack(codes, scales):
    """The values [..., d] of codes [..., d / 2] and scales [..., d / 32], in 32 bits."""
    w = codes.contiguous().view(torch.int32)
    shift = torch.tensor([[4 * i, 16 + 4 * i] for i in range(4)], dtype=torch.int32, device=codes.device)
    c = ((w[..., None, None] >> shift) & 15).reshape(*scales.shape, 32)
    return ((c - 8).float() * scales.float()[..., None]).reshape(*scales.shape[:-1], -1)


def _views(c, raw, n_blocks):
    """Codes and scales of a 4-bit array."""
    rows = n_blocks * c["layers"] * c["heads_kv"] * c["block"]
    codes = raw[:rows * c["dim"] // 2].view(n_blocks, c["layers"], c["heads_kv"], c["block"], c["dim"] // 2)
    scales = raw[rows * c["dim"] // 2:].view(torch.float16).view(n_blocks, c["layers"], c["heads_kv"], c["dim"] // 32, c["block"])
    return codes, scales


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    order = torch.randperm(c["seqs"], generator=host)
    lens, news = torch.tensor(_lens(c))[order], torch.tensor(_news(c))[order]
    n_blocks = _slots(c) // c["block"]
    ids = torch.randperm(n_blocks, generator=host).to(torch.int32)
    pages = (lens + c["block"] - 1) // c["block"]
    # blocks in no order; entries that a sequence does not need hold no block's number
    table = torch.full((c["seqs"], int(pages.max())), -1, dtype=torch.int32)
    table[torch.arange(table.shape[1])[None, :] < pages[:, None]] = ids[:int(pages.sum())]
    s = {"case": c, "n_blocks": n_blocks, "max_new": int(news.max()), "max_len": int(lens.max()), "n_tokens": int(news.sum()),
         "table": table.cuda(), "lens": lens.to(torch.int32).cuda(), "layer": c["layers"] - 1, "scale": 1 / math.sqrt(c["dim"])}
    s["starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), news.cumsum(0)]).to(torch.int32).cuda()
    shape = (n_blocks, c["layers"], c["heads_kv"], c["block"], c["dim"])
    for name in ("k", "v"):
        x = normal(*shape)
        if c["op"] == "select" and name == "k":
            x.mul_(0.6).add_(normal(*shape[:3], 1, shape[-1]))
        if c["type"] == "q4_0":
            codes, scales = _pack(x)
            s[name] = torch.cat([codes.reshape(-1), scales.transpose(-1, -2).contiguous().reshape(-1).view(torch.uint8)])
        else:
            s[name] = x.half() if c["type"] == "f16" else x
    heads = c["heads"] if c["op"] in ("append", "attend", "select") else 0
    if heads:
        s["q"] = normal(s["n_tokens"], heads, c["dim"])
        s["out"] = torch.zeros_like(s["q"])
    if c["op"] == "append":
        s["new_k"], s["new_v"] = (normal(s["n_tokens"], c["heads_kv"], c["dim"]) for _ in range(2))
        s["back_k"], s["back_v"] = torch.zeros_like(s["new_k"]), torch.zeros_like(s["new_v"])
        seq = torch.repeat_interleave(torch.arange(c["seqs"]), news)
        place = torch.arange(s["n_tokens"]) - torch.cat([torch.zeros(1, dtype=torch.int64), news.cumsum(0)])[seq] + (lens - news)[seq]
        s["positions"] = (place + c["offset"]).to(torch.int32).cuda()
        angle = torch.arange(s["max_len"] + c["offset"], device="cuda", dtype=torch.float64)[:, None] \
            * torch.pow(torch.tensor(500000.0, dtype=torch.float64, device="cuda"),
                        torch.arange(c["rot"] // 2, device="cuda", dtype=torch.float64) * (-2.0 / c["rot"]))
        s["angles"] = torch.stack([angle.cos(), angle.sin()], -1).float()
    if c["op"] in ("bounds", "select"):
        kind = torch.float32 if c["type"] == "f32" else torch.float16
        s["bounds"] = torch.zeros(n_blocks, c["layers"], c["heads_kv"], 2, c["dim"], dtype=kind, device="cuda")
    if c["op"] == "select":
        x = s["k"] if c["type"] != "q4_0" else _whole(s, "k")
        there = torch.zeros(n_blocks, dtype=torch.int64)  # positions that a block holds
        for b in range(c["seqs"]):
            at = table[b, :int(pages[b])].long()
            there[at] = (lens[b] - torch.arange(int(pages[b])) * c["block"]).clamp(max=c["block"])
        held = (torch.arange(c["block"])[None, :] < there[:, None]).cuda()[:, None, None, :, None]
        s["bounds"][:, :, :, 0] = x.masked_fill(~held, math.inf).amin(-2)
        s["bounds"][:, :, :, 1] = x.masked_fill(~held, -math.inf).amax(-2)
        s["chosen"] = torch.zeros(s["n_tokens"], c["heads_kv"], c["select"], dtype=torch.int32, device="cuda")
    return s


def _whole(s, name):
    """A 4-bit array's values, all of them."""
    codes, scales = _views(s["case"], s[name], s["n_blocks"])
    return _unpack(codes, scales.transpose(-1, -2))


# ------------------------------------------------------------------ the framework's calls
_gpu_handle = None


def _gpu():
    """The program's executor."""
    global _gpu_handle
    if _gpu_handle is None:
        _gpu_handle = importlib.import_module("llama-rust_amd").HipGemv(0)
    return _gpu_handle


def _descriptions(s):
    """The cache, the sequences and the rotation as the entry points take them: what a program keeps as long as its buffers stay."""
    if "cache" not in s:
        pkg, c = importlib.import_module("llama-rust_amd"), s["case"]
        kind = {"f32": pkg.F32, "f16": pkg.F16, "q4_0": pkg.Q4_0}[c["type"]]
        s["cache"] = pkg.KvCache(kind, c["layers"], c["heads_kv"], c["dim"], c["block"], s["n_blocks"], s["k"].data_ptr(), s["v"].data_ptr())
        one_each = s["max_new"] == 1
        s["seqs"] = pkg.KvSeqs(c["seqs"], s["table"].data_ptr(), s["table"].shape[1], s["lens"].data_ptr(), s["max_len"],
                               0 if one_each else s["starts"].data_ptr(), s["n_tokens"], s["max_new"])
        if c["op"] == "append":
            s["rope"] = pkg.Rope(s["angles"].data_ptr(), c["rot"] // 2, s["angles"].shape[0], c["rot"], halves=c["halves"],
                                 positions_ptr=s["positions"].data_ptr() if c["offset"] else 0)
    return s["cache"], s["seqs"]


def _own_run(s):
    c, gpu = s["case"], _gpu()
    cache, seqs = _descriptions(s)
    if c["op"] == "append":
        gpu.kv_append_device(cache, seqs, s["layer"], s["rope"], c["heads"], s["q"].data_ptr(), s["out"].data_ptr(), s["new_k"].data_ptr(),
                             s["new_v"].data_ptr())
        if c["type"] != "q4_0":
            return s["out"], s["k"], s["v"]
        gpu.kv_load_device(cache, seqs, s["layer"], s["back_k"].data_ptr(), s["back_v"].data_ptr())
        return s["out"], s["back_k"], s["back_v"]
    if c["op"] == "bounds":
        gpu.kv_bounds_device(cache, seqs, s["layer"], s["bounds"].data_ptr())
        return s["bounds"]
    if c["op"] == "select":
        gpu.attn_select_device(cache, seqs, s["layer"], c["heads"], s["bounds"].data_ptr(), c["select"], c["first"], c["recent"],
                               s["q"].data_ptr(), s["out"].data_ptr(), s["scale"], chosen_ptr=s["chosen"].data_ptr())
        return s["out"], s["chosen"]
    gpu.attn_device(cache, seqs, s["layer"], c["heads"], s["q"].data_ptr(), s["out"].data_ptr(), s["scale"], window=c["window"],
                    sinks=c["sinks"])
    return s["out"]


# ------------------------------------------------------------------ the plain form
def _rows_of(s, name, block, place):
    """K or V of the layer at positions given by their blocks and places there, in 32 bits: [..., key-value head, size]."""
    if s["case"]["type"] != "q4_0":
        return s[name][block, s["layer"], :, place].float()
    codes, scales = _views(s["case"], s[name], s["n_blocks"])
    return _unpack(codes[block, s["layer"], :, place], scales[block, s["layer"], :, :, place])


def _new_rows(s):
    """Sequence, block and place of every new token."""
    c = s["case"]
    starts, lens = s["starts"].long(), s["lens"].long()
    row = torch.arange(s["n_tokens"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    t = lens[seq] - starts[seq + 1] + row
    return seq, t, s["table"].long()[seq, t // c["block"]], t % c["block"]


def _turned(s, x):
    """Rows [tokens, heads, size] turned by their positions, in 64 bits, rounded once."""
    c = s["case"]
    cs = s["angles"][s["positions"].long()].double()[:, None]
    y, h = x.double().clone(), c["rot"] // 2
    a, b = (y[..., :h].clone(), y[..., h:2 * h].clone()) if c["halves"] else (y[..., 0:2 * h:2].clone(), y[..., 1:2 * h:2].clone())
    at_a, at_b = (slice(0, h), slice(h, 2 * h)) if c["halves"] else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
    y[..., at_a] = a * cs[..., 0] - b * cs[..., 1]
    y[..., at_b] = a * cs[..., 1] + b * cs[..., 0]
    return y.float()


def _plain_append(s):
    c = s["case"]
    _, _, block, place = _new_rows(s)
    q, k = _turned(s, s["q"]), _turned(s, s["new_k"])
    if c["type"] != "q4_0":
        s["k"][block, s["layer"], :, place] = k.to(s["k"].dtype)
        s["v"][block, s["layer"], :, place] = s["new_v"].to(s["v"].dtype)
        return q, s["k"], s["v"]
    for name, x in (("k", k), ("v", s["new_v"])):
        codes, scales = _views(c, s[name], s["n_blocks"])
        codes[block, s["layer"], :, place], scales[block, s["layer"], :, :, place] = _pack(x)
    return q, _rows_of(s, "k", block, place), _rows_of(s, "v", block, place)


def _plain_attend(s):
    c = s["case"]
    n, m, length, kv, d = c["seqs"], s["max_new"], s["max_len"], c["heads_kv"], c["dim"]
    starts, lens = s["starts"].long(), s["lens"].long()
    news = starts[1:] - starts[:-1]
    t = torch.arange(length, device="cuda")
    there = t[None, :] < lens[:, None]
    block = s["table"].long()[:, t // c["block"]].clamp(min=0)
    place = (t % c["block"])[None].expand(n, length)
    k = _rows_of(s, "k", block, place).permute(0, 2, 1, 3).contiguous()  # [seqs, kv heads, positions, size]
    v = _rows_of(s, "v", block, place).permute(0, 2, 1, 3).contiguous()
    i = torch.arange(m, device="cuda")
    real = i[None, :] < news[:, None]
    rows = (starts[:-1, None] + i[None, :]).clamp(max=s["n_tokens"] - 1)
    q = s["q"][rows].view(n, m, kv, -1, d).permute(0, 2, 1, 3, 4)  # [seqs, kv heads, tokens, heads of one, size]
    group = q.shape[3]
    score = torch.matmul(q.reshape(n, kv, m * group, d), k.transpose(2, 3).contiguous()).view(n, kv, m, group, length).mul_(s["scale"])
    p = (lens - news)[:, None, None] + i[None, :, None]
    sees = there[:, None, :] & (t <= p) & real[:, :, None]
    if c["window"]:
        sees &= (p - t < c["window"]) | (t < c["sinks"])
    score.masked_fill_(~sees[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = e.sum(-1, keepdim=True, dtype=torch.float64).float()
    e /= torch.where(total > 0, total, torch.ones_like(total))
    out = torch.empty_like(s["q"])
    o = torch.matmul(e.view(n, kv, m * group, length), v).view(n, kv, m, group, d).permute(0, 2, 1, 3, 4).reshape(n, m, kv * group, d)
    out[rows[real]] = o[real]
    return out


def _plain_bounds(s):
    c = s["case"]
    lens, starts = s["lens"].long(), s["starts"].long()
    news = starts[1:] - starts[:-1]
    first = (lens - news) // c["block"]
    most = (s["max_new"] - 1) // c["block"] + 2
    j = first[:, None] + torch.arange(most, device="cuda")[None]
    real = j * c["block"] < lens[:, None]
    block = torch.gather(s["table"].long(), 1, j.clamp(max=s["table"].shape[1] - 1))[real]
    held = torch.arange(c["block"], device="cuda")[None] < (lens[:, None] - j * c["block"])[real][:, None]
    place = torch.arange(c["block"], device="cuda")[None].expand(block.shape[0], -1)
    x = _rows_of(s, "k", block[:, None].expand(place.shape), place)  # [blocks, positions, kv heads, size]
    s["bounds"][block, s["layer"], :, 0] = x.masked_fill(~held[..., None, None], math.inf).amin(1).to(s["bounds"].dtype)
    s["bounds"][block, s["layer"], :, 1] = x.masked_fill(~held[..., None, None], -math.inf).amax(1).to(s["bounds"].dtype)
    return s["bounds"]


def _plain_select(s):
    c = s["case"]
    kv, d, most = c["heads_kv"], c["dim"], c["select"]
    seq, p, _, _ = _new_rows(s)
    tokens = seq.shape[0]
    pages = -(-s["max_len"] // c["block"])
    blocks = s["table"].long()[:, :pages].clamp(min=0)
    lo, hi = (s["bounds"][blocks, s["layer"], :, w].double().permute(0, 2, 3, 1).contiguous() for w in (0, 1))  # [seqs, kv, size, blocks]
    q = s["q"].view(tokens, kv, -1, d)
    # a sequence's tokens together, so that its bounds are multiplied once
    news = (s["starts"][1:] - s["starts"][:-1]).long()
    row = torch.arange(tokens, device="cuda") - s["starts"].long()[seq]
    padded = torch.zeros(c["seqs"], s["max_new"], *q.shape[1:], dtype=torch.float64, device="cuda")
    padded[seq, row] = q.double()
    padded = padded.permute(0, 2, 1, 3, 4).reshape(c["seqs"], kv, -1, d)
    bound = torch.matmul(padded.clamp(min=0), hi) + torch.matmul(padded.clamp(max=0), lo)
    score = bound.view(c["seqs"], kv, s["max_new"], -1, pages).amax(3).permute(0, 2, 1, 3)[seq, row].float()  # [tokens, kv, blocks]
    j = torch.arange(pages, device="cuda")
    last = (p // c["block"])[:, None, None]
    always = (j < c["first"]) | (j > last - c["recent"])
    key = torch.where(always, torch.full_like(score, math.inf), score)
    key = torch.where(j <= last, key, torch.full_like(score, -math.inf))
    kept = min(most, pages)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :kept]
    best = torch.where(torch.arange(kept, device="cuda") <= last, best, torch.full_like(best, pages)).sort(-1).values  # [tokens, kv, kept]
    chosen = torch.full((tokens, kv, most), -1, dtype=torch.int32, device="cuda")
    chosen[..., :kept] = torch.where(best < pages, best, torch.full_like(best, -1)).to(torch.int32)
    t = (best[..., None] * c["block"] + torch.arange(c["block"], device="cuda")).view(tokens, kv, -1)
    sees = (best < pages).repeat_interleave(c["block"], -1) & (t <= p[:, None, None])
    block = s["table"].long()[seq[:, None, None], (t // c["block"]).clamp(max=pages - 1)].clamp(min=0)
    head = torch.arange(kv, device="cuda")[None, :, None].expand(t.shape)
    place = t % c["block"]

    def rows(name):
        if c["type"] != "q4_0":
            return s[name][block, s["layer"], head, place].float()
        codes, scales = _views(c, s[name], s["n_blocks"])
        return _unpack(codes[block, s["layer"], head, place], scales[block, s["layer"], head, :, place])

    x = torch.matmul(q.contiguous(), rows("k").transpose(2, 3).contiguous()).mul_(s["scale"])  # [tokens, kv, heads of one, positions]
    x.masked_fill_(~sees[:, :, None, :], -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    x /= x.sum(-1, keepdim=True, dtype=torch.float64).float()
    return torch.matmul(x, rows("v")).view(s["q"].shape), chosen


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "attend": _plain_attend, "bounds": _plain_bounds, "select": _plain_select}[state["case"]["op"]](state)


# ------------------------------------------------------------------ from the definition, in 64 bits
def _four_bits(x):
    """What a 4-bit cache makes of rows [..., size] of f32 numbers."""
    b = x.reshape(*x.shape[:-1], -1, 32).double()
    most, _ = b.abs().max(-1, keepdim=True)
    is_most = (b.abs() == most).int()
    largest = (b * (is_most * (is_most.cumsum(-1) == 1))).sum(-1, keepdim=True)
    m, e = torch.frexp(largest / -8)
    d = torch.ldexp(torch.round(m * 256), e - 8).clamp(-8160, 8160)  # eight significant bits
    d = torch.round(d * 2.0 ** 24) / 2.0 ** 24  # f16's smallest step
    codes = torch.where(d == 0, torch.zeros_like(b), torch.round(b / d)).clamp(-8, 7)
    return (codes * d).reshape(x.shape)


def _cached(s, name, b, n, head):
    """K or V of a sequence's first n positions of one key-value head, in 64 bits."""
    c = s["case"]
    t = torch.arange(n, device="cuda")
    block, place = s["table"][b].long()[t // c["block"]], t % c["block"]
    if c["type"] != "q4_0":
        return s[name][block, s["layer"], head, place].double()
    rows = s["n_blocks"] * c["layers"] * c["heads_kv"] * c["block"]
    row = ((block * c["layers"] + s["layer"]) * c["heads_kv"] + head) * c["block"] + place
    bytes_of = s[name][:rows * c["dim"] // 2].view(rows, c["dim"] // 2)[row].long()
    unit = (row // c["block"])[:, None] * (c["dim"] // 32) + torch.arange(c["dim"] // 32, device="cuda")[None]
    scale = s[name][rows * c["dim"] // 2:].view(torch.float16)[unit * c["block"] + place[:, None]].double()
    e = torch.arange(c["dim"], device="cuda")
    bit = e % 8 // 2 * 4 + e % 2 * 16
    nibble = (bytes_of[:, e // 8 * 4 + bit // 8] >> (bit % 8)) & 15
    return (nibble - 8).double() * scale[:, e // 32]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    lens, starts, layer = s["lens"].tolist(), s["starts"].tolist(), s["layer"]
    kv, group = c["heads_kv"], c["heads"] // c["heads_kv"]
    if c["op"] == "append":
        def turn(x):
            angle = s["angles"][s["positions"].long()].double()
            pair = torch.complex(angle[..., 0], angle[..., 1])[:, None]
            y, h = x.double().clone(), c["rot"] // 2
            first = torch.arange(h, device="cuda") * (1 if c["halves"] else 2)
            second = first + (h if c["halves"] else 1)
            z = torch.complex(y[..., first], y[..., second]) * pair
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q, k = turn(s["q"]), turn(s["new_k"])
        if c["type"] == "q4_0":
            return q, _four_bits(k.float()), _four_bits(s["new_v"])
        all_k, all_v = s["k"].double(), s["v"].double()
        for b in range(c["seqs"]):
            n = starts[b + 1] - starts[b]
            t = torch.arange(lens[b] - n, lens[b], device="cuda")
            block, place = s["table"][b].long()[t // c["block"]], t % c["block"]
            all_k[block, layer, :, place] = k[starts[b]:starts[b + 1]]
            all_v[block, layer, :, place] = s["new_v"][starts[b]:starts[b + 1]].double()
        return q, all_k, all_v
    if c["op"] == "bounds":
        bounds = s["bounds"].double()
        for b in range(c["seqs"]):
            n = starts[b + 1] - starts[b]
            for h in range(kv):
                x = _cached(s, "k", b, lens[b], h)
                for j in range((lens[b] - n) // c["block"], (lens[b] - 1) // c["block"] + 1):
                    keys = x[j * c["block"]:(j + 1) * c["block"]]
                    bounds[int(s["table"][b, j]), layer, h, 0] = keys.min(0).values
                    bounds[int(s["table"][b, j]), layer, h, 1] = keys.max(0).values
        return bounds
    if c["op"] == "select" and s["n_tokens"] * kv > 4000:
        return None  # a loop over tokens and heads
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    chosen = torch.full((s["n_tokens"], kv, c.get("select", 0)), -1, dtype=torch.int32, device="cuda")
    for b in range(c["seqs"]):
        n = starts[b + 1] - starts[b]
        t = torch.arange(lens[b], device="cuda")
        p = torch.arange(lens[b] - n, lens[b], device="cuda")[:, None]
        for h in range(kv):
            k, v = _cached(s, "k", b, lens[b], h), _cached(s, "v", b, lens[b], h)
            hidden = (t > p)
            if c["op"] == "attend" and c["window"]:
                hidden = hidden | ((t <= p - c["window"]) & (t >= c["sinks"]))
            if c["op"] == "select":
                pages = s["table"][b, :-(-lens[b] // c["block"])].long()
                lo, hi = s["bounds"][pages, layer, h, 0].double(), s["bounds"][pages, layer, h, 1].double()
                for i in range(n):
                    mine = s["q"][starts[b] + i, h * group:(h + 1) * group].double()
                    last = (lens[b] - n + i) // c["block"]
                    kept = torch.arange(last + 1, device="cuda")
                    if last + 1 > c["select"]:
                        best = torch.maximum(mine[:, None] * hi[:last + 1], mine[:, None] * lo[:last + 1]).sum(-1).amax(0).float()
                        middle = best[c["first"]:last + 1 - c["recent"]]
                        by_score = torch.argsort(-middle, stable=True)[:c["select"] - c["first"] - c["recent"]] + c["first"]
                        kept = torch.cat([kept[:c["first"]], by_score.sort().values, kept[last + 1 - c["recent"]:]])
                    chosen[starts[b] + i, h, :kept.shape[0]] = kept.to(torch.int32)
                    hidden[i] |= ~torch.isin(t // c["block"], kept)
            for g in range(group):
                q = s["q"][starts[b]:starts[b + 1], h * group + g].double()
                x = (q @ k.t().contiguous()) * s["scale"]
                out[starts[b]:starts[b + 1], h * group + g] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
    return (out, chosen) if c["op"] == "select" else out
