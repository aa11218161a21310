"""What the operators over a paged key-value cache are measured on: storing new rows, attention that reads the cache, eviction.

The cache is two arrays [block][layer][key-value head][position in the block][head size] of f32 or f16 and, where weights are
kept, a third one without the last axis. A sequence's position t lies in block table[t // kv_block]. `lens` counts a
sequence's cached positions, the new ones among them: new row i of n stands at position len - n + i.

  store    K and V of new tokens into the cache, rounded to its type
  attend   softmax(scale q K^T) V for every new token: token p sees t <= p, with a window only the last `window` positions and
           the first `sinks`; with `weights` each key-value head's accumulated weight of every position becomes decay times
           what it was plus the probabilities that this call's tokens and query heads gave it
  evict    keeps `keep` positions of each sequence, per layer and key-value head: the first `first`, the last `recent`, and of
           those between them the heaviest (ties to the lower position), in their order, in the blocks of another table

Queries, keys and values are N(0, 1) as projections after a norm are; accumulated weights have a few heavy positions, a
long tail and exact zeros, as sums of softmax rows in f32 have.
"""
import importlib
import math

import torch

own = False

# Most bytes and operations of a drawn pass: below the largest listed case's.
MOST_BYTES, MOST_FLOPS = 4.0e8, 2.0e11


def listed():
    return [
        # one user's next token: 8 rows of K and V, where only the call counts
        {"name": "store_1_token", "op": "store", "type": "f32", "heads": 32, "heads_kv": 8, "dim": 128, "block": 16, "layers": 2,
         "seqs": 1, "new": 1, "len": 130},
        # a prompt chunk of the device session's largest size into an f16 cache
        {"name": "store_512_tokens", "op": "store", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 16, "layers": 2,
         "seqs": 1, "new": 512, "len": 900},
        # chat with one user, an 8B model, a short history: the smallest attention
        {"name": "decode_1_short", "op": "attend", "type": "f32", "heads": 32, "heads_kv": 8, "dim": 128, "block": 16, "layers": 2,
         "seqs": 1, "new": 1, "len": 200, "window": 0, "sinks": 0, "weights": False},
        # one user, a whole book in the cache: few rows, a long axis
        {"name": "decode_1_long", "op": "attend", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 64, "layers": 2,
         "seqs": 1, "new": 1, "len": 100003, "window": 0, "sinks": 0, "weights": False},
        # a server's step with a half-billion-parameter model (width 896): sequences of every length, seven query heads a key
        {"name": "decode_32_ragged", "op": "attend", "type": "f32", "heads": 14, "heads_kv": 2, "dim": 64, "block": 16, "layers": 2,
         "seqs": 32, "new": 1, "len": 8192, "window": 0, "sinks": 0, "weights": False},
        # endless streams: a window of the last positions and the first four, whatever the length
        {"name": "decode_8_window", "op": "attend", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 32, "layers": 2,
         "seqs": 8, "new": 1, "len": 32768, "window": 4096, "sinks": 4, "weights": False},
        # a long document's next chunk: bound by the matrix cores
        {"name": "chunk_2048", "op": "attend", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 64, "layers": 2,
         "seqs": 1, "new": 2048, "len": 8192, "window": 0, "sinks": 0, "weights": False},
        # several prompts at once, none a whole tile, a head size and blocks that are no powers of two, a window inside them
        {"name": "chunk_ragged_window", "op": "attend", "type": "f16", "heads": 24, "heads_kv": 4, "dim": 80, "block": 20, "layers": 2,
         "seqs": 5, "new": 401, "len": 1201, "window": 300, "sinks": 4, "weights": False},
        # a server's step that keeps the weights an eviction goes by
        {"name": "decode_16_weights", "op": "attend", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 16, "layers": 2,
         "seqs": 16, "new": 1, "len": 4096, "window": 0, "sinks": 0, "weights": True},
        # a prompt chunk in an f32 cache, the session's default, with the weights
        {"name": "chunk_512_weights", "op": "attend", "type": "f32", "heads": 32, "heads_kv": 8, "dim": 128, "block": 16, "layers": 2,
         "seqs": 1, "new": 512, "len": 512, "window": 0, "sinks": 0, "weights": True},
        # one user's cache back to its budget: one layer, few workgroups
        {"name": "evict_1", "op": "evict", "type": "f32", "heads": 32, "heads_kv": 8, "dim": 128, "block": 16, "layers": 2, "seqs": 1,
         "len": 1200, "keep": 1001, "first": 4, "recent": 128},
        # a server's caches halved: the rows that stay are most of the work
        {"name": "evict_8", "op": "evict", "type": "f16", "heads": 32, "heads_kv": 8, "dim": 128, "block": 32, "layers": 4, "seqs": 8,
         "len": 8192, "keep": 4096, "first": 4, "recent": 512},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv = rng.choice([1, 2, 4, 8])
    c = {"op": rng.choice(["store", "attend", "attend", "attend", "attend", "evict"]), "type": rng.choice(["f32", "f16"]),
         "heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "heads_kv": kv, "dim": rng.choice([40, 64, 64, 80, 96, 128, 128, 128, 192, 256]),
         "block": rng.choice([1, 16, 16, 20, 32, 64, 128]), "layers": rng.choice([1, 2, 3]), "seqs": _log(rng, 1, 64)}
    if c["op"] == "evict":
        c.update(len=_log(rng, 40, 16384), first=rng.choice([0, 4]), recent=rng.choice([0, 1, 16]))
        c["keep"] = max(c["first"] + c["recent"] + 1, int(c["len"] * rng.uniform(0.2, 0.95)))
    else:
        c["new"] = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 1024)])
        c["len"] = c["new"] + _log(rng, 1, 65536 if c["seqs"] <= 4 and c["new"] < 16 else 8192)
    if c["op"] == "attend":
        c["window"] = rng.choice([0, 0, _log(rng, 16, 4096)])
        c["sinks"] = rng.choice([0, 4]) if c["window"] else 0
        c["weights"] = rng.random() < 0.25
    # fewer, then shorter sequences until the pass fits
    while _cost(c) > 1.0:
        if c["seqs"] > 1:
            c["seqs"] = (c["seqs"] + 1) // 2
        elif c["op"] == "evict":
            c["len"], c["keep"] = c["len"] // 2, max(c["first"] + c["recent"] + 1, c["keep"] // 2)
        else:
            c["new"] = (c["new"] + 1) // 2
            c["len"] = max(c["new"] + 1, c["len"] // 2)
    return c


def _cost(c):
    w = work(c)
    return max(w["bytes"] / MOST_BYTES, w["flops"] / MOST_FLOPS, _slots(c) * c["layers"] * c["heads_kv"] * c["dim"] / 8.0e8)


# ------------------------------------------------------------------ shapes: the lengths follow from the case, their order from the seed
def _lens(c):
    """Cached positions of every sequence, spread evenly up to the longest."""
    n, least = c["seqs"], c.get("new", 1)
    return [least + (c["len"] - least) * (b + 1) // n for b in range(n)]


def _news(c):
    """New tokens of every sequence: as many for each, except that the chunks of several prompts differ."""
    n, most = c["seqs"], c.get("new", 0)
    return [most] * n if most <= 1 else [max(1, most * (b + 1) // n) for b in range(n)]


def _kept(c):
    return [min(x, c["keep"]) for x in _lens(c)]


def _slots(c):
    pages = sum(-(-x // c["block"]) for x in _lens(c))
    if c["op"] == "evict":
        pages += sum(-(-x // c["block"]) for x in _kept(c))
    return (pages + 3) * c["block"]


def _visible(c):
    """Pairs of a token and a position it sees, and positions that any token of the call sees."""
    pairs = seen = 0
    for length, new in zip(_lens(c), _news(c)):
        first, w, k = length - new, c["window"], c["sinks"]
        if not w:
            pairs += new * first + new * (new + 1) // 2
            seen += length
            continue
        edge = first + 1 - w  # the first position in the first token's window
        seen += length - max(0, edge - min(k, max(0, edge)))
        full = min(new, max(0, w - first))  # tokens whose window reaches the start
        pairs += full * first + full * (full + 1) // 2
        rest = new - full
        pairs += rest * w
        for i in ((full, new) if rest else ()):  # sinks before the window: they grow until there are k of them
            m = first + i + 1 - w if i == full else first + new - w
            pairs += 0 if i == full else _sum_min(first + full + 1 - w, m, k)
    return pairs, seen


def _sum_min(a, b, k):
    """Sum of min(x, k) for x in a .. b."""
    low = max(0, min(b, k) - a + 1)
    return low * (a + a + low - 1) // 2 + (b - a + 1 - low) * k


def work(case):
    c = case
    size, kv = 2 if c["type"] == "f16" else 4, c["heads_kv"]
    tables = 4 * sum(-(-x // c["block"]) for x in _lens(c))
    if c["op"] == "store":
        values = 2 * sum(_news(c)) * kv * c["dim"]
        return {"bytes": values * (4 + size) + tables, "flops": 0}
    if c["op"] == "evict":
        rows = c["layers"] * kv * sum(_kept(c))
        return {"bytes": 4 * c["layers"] * kv * sum(_lens(c)) + rows * (4 * c["dim"] * size + 4) + 2 * tables, "flops": 0}
    pairs, seen = _visible(c)
    sums = 8 * kv * sum(_lens(c)) if c["weights"] else 0
    return {"bytes": 2 * seen * kv * c["dim"] * size + 8 * sum(_news(c)) * c["heads"] * c["dim"] + sums + tables,
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    dt = torch.float16 if c["type"] == "f16" else torch.float32

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    order = torch.randperm(c["seqs"], generator=host)
    lens, news = torch.tensor(_lens(c))[order], torch.tensor(_news(c))[order]
    kept = torch.tensor(_kept(c))[order] if c["op"] == "evict" else None
    n_blocks = _slots(c) // c["block"]
    ids = torch.randperm(n_blocks, generator=host).to(torch.int32)

    def table(of, at):
        """Blocks in no order; entries that a sequence does not need hold no block's number."""
        pages = (of + c["block"] - 1) // c["block"]
        t = torch.full((c["seqs"], int(pages.max())), -1, dtype=torch.int32)
        used = torch.arange(t.shape[1])[None, :] < pages[:, None]
        t[used] = ids[at:at + int(pages.sum())]
        return t.cuda(), at + int(pages.sum())

    s = {"case": c, "n_blocks": n_blocks, "max_new": int(news.max()), "max_len": int(lens.max()), "n_tokens": int(news.sum())}
    s["table"], used = table(lens, 0)
    s["lens"] = lens.to(torch.int32).cuda()
    shape = (n_blocks, c["layers"], c["heads_kv"], c["block"], c["dim"])
    s["k"], s["v"] = (torch.empty(shape, dtype=dt, device="cuda").normal_(generator=gen) for _ in range(2))
    s["layer"] = c["layers"] - 1
    if c["op"] == "evict":
        s["to"], _ = table(kept, used)
        s["w"] = torch.exp(2 * normal(*shape[:-1])).sub_(0.1).clamp_(min=0)
        s["new_lens"] = torch.zeros(c["seqs"], dtype=torch.int32, device="cuda")
        return s
    s["starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), news.cumsum(0)]).to(torch.int32).cuda()
    if c["op"] == "store":
        s["new_k"], s["new_v"] = (normal(s["n_tokens"], c["heads_kv"], c["dim"]) for _ in range(2))
        return s
    s["q"] = normal(s["n_tokens"], c["heads"], c["dim"])
    s["out"] = torch.zeros_like(s["q"])
    s["scale"] = 1 / math.sqrt(c["dim"])
    s["w"] = torch.zeros(shape[:-1], device="cuda") if c["weights"] else None
    return s


# ------------------------------------------------------------------ the framework's calls
_gpu_handle = None


def _gpu():
    """The program's executor."""
    global _gpu_handle
    if _gpu_handle is None:
        _gpu_handle = importlib.import_module("llama-rust_amd").HipGemv(0)
    return _gpu_handle


def _descriptions(s):
    """The cache and the sequences as the entry points take them: what a program keeps as long as its buffers stay."""
    if "cache" not in s:
        pkg, c = importlib.import_module("llama-rust_amd"), s["case"]
        s["cache"] = pkg.KvCache(pkg.F16 if c["type"] == "f16" else pkg.F32, c["layers"], c["heads_kv"], c["dim"], c["block"], s["n_blocks"],
                                 s["k"].data_ptr(), s["v"].data_ptr(), s["w"].data_ptr() if s.get("w") is not None else 0)
        one_each = c["op"] == "evict" or s["max_new"] == 1
        s["seqs"] = pkg.KvSeqs(c["seqs"], s["table"].data_ptr(), s["table"].shape[1], s["lens"].data_ptr(), s["max_len"],
                               0 if one_each else s["starts"].data_ptr(), c["seqs"] if one_each else s["n_tokens"],
                               1 if one_each else s["max_new"])
    return s["cache"], s["seqs"]


def _own_run(s):
    c, gpu = s["case"], _gpu()
    cache, seqs = _descriptions(s)
    if c["op"] == "store":
        gpu.kv_store_device(cache, seqs, s["layer"], s["new_k"].data_ptr(), s["new_v"].data_ptr())
        return s["k"], s["v"]
    if c["op"] == "evict":
        gpu.kv_evict_device(cache, seqs, 0, c["layers"], c["keep"], c["first"], c["recent"], s["to"].data_ptr(), s["to"].shape[1],
                            s["new_lens"].data_ptr())
        return s["k"], s["v"], s["w"], s["new_lens"]
    gpu.attn_device(cache, seqs, s["layer"], c["heads"], s["q"].data_ptr(), s["out"].data_ptr(), s["scale"], window=c["window"],
                    sinks=c["sinks"], weights=c["weights"], decay=0.0)
    return (s["out"], s["w"]) if c["weights"] else s["out"]


# ------------------------------------------------------------------ the plain form
def _rows(c, table, t):
    """Where the positions t [seqs, n] lie: block and place in it."""
    return torch.gather(table.long(), 1, (t // c["block"]).clamp(max=table.shape[1] - 1)), t % c["block"]


def _plain_store(s):
    c = s["case"]
    starts, lens = s["starts"].long(), s["lens"].long()
    row = torch.arange(s["n_tokens"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    t = lens[seq] - starts[seq + 1] + row
    block, place = s["table"].long()[seq, t // c["block"]], t % c["block"]
    s["k"][block, s["layer"], :, place] = s["new_k"].to(s["k"].dtype)
    s["v"][block, s["layer"], :, place] = s["new_v"].to(s["v"].dtype)
    return s["k"], s["v"]


def _plain_attend(s):
    c = s["case"]
    n, m, length, kv, d = c["seqs"], s["max_new"], s["max_len"], c["heads_kv"], c["dim"]
    starts, lens = s["starts"].long(), s["lens"].long()
    news = starts[1:] - starts[:-1]
    t = torch.arange(length, device="cuda")
    there = t[None, :] < lens[:, None]
    block, place = _rows(c, s["table"], t[None, :].expand(n, length))
    block = block.clamp(min=0)
    k = s["k"][block, s["layer"], :, place].float().permute(0, 2, 1, 3).contiguous()  # [seqs, kv heads, positions, size]
    v = s["v"][block, s["layer"], :, place].float().permute(0, 2, 1, 3).contiguous()
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
    if not c["weights"]:
        return out
    w = e.sum((2, 3), dtype=torch.float64).float().permute(0, 2, 1)  # [seqs, positions, kv heads]
    s["w"][block[there], s["layer"], :, place[there]] = w[there]
    return out, s["w"]


def _plain_evict(s):
    c = s["case"]
    n, length, keep = c["seqs"], s["max_len"], c["keep"]
    lens = s["lens"].long()
    t = torch.arange(length, device="cuda")[None, :].expand(n, length)
    block, place = _rows(c, s["table"], t)
    w = s["w"][block.clamp(min=0), :, :, place].permute(0, 2, 3, 1)  # [seqs, layers, kv heads, positions]
    always = (t < c["first"]) | (t >= lens[:, None] - c["recent"])
    key = torch.where(always[:, None, None], torch.full_like(w, math.inf), w)
    key = torch.where((t < lens[:, None])[:, None, None], key, torch.full_like(w, -math.inf))
    new = lens.clamp(max=keep)
    most = min(keep, length)
    best = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :most]
    rank = torch.arange(most, device="cuda")
    best = torch.where(rank < new[:, None, None, None], best, torch.full_like(best, length)).sort(-1).values  # kept ones first, ascending
    stays = (rank[None] < new[:, None])[:, None, None].expand(best.shape)
    at = torch.nonzero(stays, as_tuple=True)
    seq, layer, head, r = at
    old = best[at]
    to = torch.gather(s["to"].long(), 1, (torch.arange(most, device="cuda") // c["block"])[None].expand(n, most))[seq, r]
    src = (block[seq, old], layer, head, place[seq, old])
    dst = (to, layer, head, r % c["block"])
    for x in (s["k"], s["v"], s["w"]):
        x[dst] = x[src]
    s["new_lens"].copy_(new)
    return s["k"], s["v"], s["w"], s["new_lens"]


def run(state):
    if own:
        return _own_run(state)
    return {"store": _plain_store, "attend": _plain_attend, "evict": _plain_evict}[state["case"]["op"]](state)


# ------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    lens, table, layer = s["lens"].tolist(), s["table"].tolist(), s["layer"]

    def where(b, n, tab):
        """Blocks and places of a sequence's first n positions."""
        t = torch.arange(n, device="cuda")
        return torch.tensor(tab[b], device="cuda")[t // c["block"]].long(), t % c["block"]

    if c["op"] == "store":
        k, v = s["k"].double(), s["v"].double()
        starts = s["starts"].tolist()
        for b in range(c["seqs"]):
            block, place = where(b, lens[b], table)
            n = starts[b + 1] - starts[b]
            block, place = block[lens[b] - n:], place[lens[b] - n:]
            k[block, layer, :, place] = s["new_k"][starts[b]:starts[b + 1]].double()
            v[block, layer, :, place] = s["new_v"][starts[b]:starts[b + 1]].double()
        return k, v
    if c["op"] == "evict":
        k, v, w, to = s["k"].double(), s["v"].double(), s["w"].double(), s["to"].tolist()
        for b in range(c["seqs"]):
            block, place = where(b, lens[b], table)
            new = min(lens[b], c["keep"])
            block_to, place_to = where(b, new, to)
            for la in range(c["layers"]):
                for h in range(c["heads_kv"]):
                    stays = torch.zeros(lens[b], dtype=torch.bool, device="cuda")
                    if lens[b] <= c["keep"]:
                        stays[:] = True
                    else:
                        stays[:c["first"]] = True
                        stays[lens[b] - c["recent"]:] = True
                        mid = w[block, la, h, place][c["first"]:lens[b] - c["recent"]]
                        # by weight, heaviest first; equal ones stay in their order
                        order = torch.argsort(-mid, stable=True)[:c["keep"] - c["first"] - c["recent"]]
                        stays[order + c["first"]] = True
                    for x in (k, v, w):
                        x[block_to, la, h, place_to] = x[block[stays], la, h, place[stays]]
        return k, v, w, torch.tensor([min(x, c["keep"]) for x in lens], dtype=torch.int32)
    starts = s["starts"].tolist()
    group = c["heads"] // c["heads_kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    w = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda") if c["weights"] else None
    for b in range(c["seqs"]):
        block, place = where(b, lens[b], table)
        n = starts[b + 1] - starts[b]
        t = torch.arange(lens[b], device="cuda")
        p = torch.arange(lens[b] - n, lens[b], device="cuda")[:, None]
        hidden = t > p
        if c["window"]:
            hidden |= (t <= p - c["window"]) & (t >= c["sinks"])
        for h in range(c["heads_kv"]):
            k, v = s["k"][block, layer, h, place].double(), s["v"][block, layer, h, place].double()
            for g in range(group):
                q = s["q"][starts[b]:starts[b + 1], h * group + g].double()
                x = (q @ k.t().contiguous()) * s["scale"]
                prob = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                out[starts[b]:starts[b + 1], h * group + g] = prob @ v
                if w is not None:
                    w[block, layer, h, place] += prob.sum(0)
    return (out, w) if w is not None else out
