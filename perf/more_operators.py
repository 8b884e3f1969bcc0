"""The operators of a decoder that goes on from one prompt in many ways, as cases to be measured.

Four kinds of case, each through the package's public entry points:

* ``prefix``: attention of a few query tokens of each sequence over the 4-bit cache, where groups of sequences share
  the pages of a long prefix;
* ``pages``: the bookkeeping of the cache's pages on the device: a decoding step (pages for new tokens, pages before a
  window given back), sequences forked (the page that a fork ends in is copied), and compaction (everything moved to
  the lowest pages);
* ``score``: the log probabilities of given tokens, the entropy, and the likeliest alternatives, of rows of logits;
* ``rotate``: the RMS norm of every query and key head and its rotation by the token's position.

The cache is a uint8 tensor [pages, kv_heads, tiles, 34 * head_dim]: a tile holds 32 tokens of one head.  A value has
4 bits (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), and 32 neighbouring values share a
power-of-two scale (a byte, exponent + 127).  A sequence's tokens are found through its row of a page table.

A pool of pages is refs (int32, how many table entries hold each page) and free (int32 words, bit p % 32 of word p / 32
is set where page p is held by none).  The lowest free page is given first.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TILE = 32
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # eight continuations of the small model's 500-token prompt, 480 of it in shared pages: latency
        {"name": "prefix 8x(480+21) 16/16x64", "kind": "prefix", "groups": 1, "batch": 8, "shared": 480, "cut": 0,
         "tail": 21, "queries": 1, "heads": 16, "kv": 16, "dim": 64, "page": 32, "dtype": "f32"},
        # 64 conversations behind one long instruction
        {"name": "prefix 64x(8000+300) 32/8x128", "kind": "prefix", "groups": 1, "batch": 64, "shared": 8000, "cut": 0,
         "tail": 300, "queries": 1, "heads": 32, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # four documents, 16 questions each, four drafted tokens at a time; the prefix ends inside a shared page
        {"name": "prefix 4x16x(3957+711) 16/4x64", "kind": "prefix", "groups": 4, "batch": 16, "shared": 3968, "cut": 11,
         "tail": 711, "queries": 4, "heads": 16, "kv": 4, "dim": 64, "page": 128, "dtype": "f16"},
        # 256 samples of one long problem
        {"name": "prefix 256x(16000+500) 32/8x128", "kind": "prefix", "groups": 1, "batch": 256, "shared": 16000,
         "cut": 0, "tail": 500, "queries": 1, "heads": 32, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one decoding step of 64 conversations with a window: pages for the new tokens, pages before the window back
        {"name": "pages step 64", "kind": "pages", "what": "step", "batch": 64, "tokens": 130000, "more": 1,
         "window": 1024, "page": 64, "pages": 4096, "kv": 8, "dim": 128, "layers": 0},
        # four prompts forked into 16 continuations each, four layers' caches
        {"name": "pages fork 4 to 64", "kind": "pages", "what": "fork", "batch": 4, "children": 64, "tokens": 8190,
         "page": 64, "pages": 512, "kv": 8, "dim": 128, "layers": 4},
        # a fragmented cache moved together before it is shrunk or sent on
        {"name": "pages compact 6000", "kind": "pages", "what": "compact", "batch": 48, "tokens": 190000, "page": 64,
         "pages": 6000, "kv": 8, "dim": 128, "layers": 1},
        # one decoding step with the 20 likeliest tokens reported
        {"name": "score 1x32000 top 20", "kind": "score", "rows": 1, "vocab": 32000, "top": 20, "dtype": "f32",
         "temperature": 1.0},
        # the small model's 500-token prompt
        {"name": "score 500x32000 top 5", "kind": "score", "rows": 500, "vocab": 32000, "top": 5, "dtype": "f32",
         "temperature": 1.0},
        # many answers scored, a large odd vocabulary
        {"name": "score 2048x100003 top 20", "kind": "score", "rows": 2048, "vocab": 100003, "top": 20, "dtype": "bf16",
         "temperature": 0.7},
        # one decoding step of 64 conversations
        {"name": "rotate step 64 32/8x128", "kind": "rotate", "batch": 64, "tokens": 64, "past": 2000, "heads": 32,
         "kv": 8, "dim": 128, "rotary": 128, "norm": True, "interleaved": False, "base": 500000.0, "dtype": "bf16",
         "fused": True},
        # prompts of odd lengths, queries and keys as parts of one projection's output
        {"name": "rotate prompts 8190 32/8x128", "kind": "rotate", "batch": 3, "tokens": 8190, "past": 0, "heads": 32,
         "kv": 8, "dim": 128, "rotary": 128, "norm": True, "interleaved": False, "base": 10000.0, "dtype": "bf16",
         "fused": True},
    ]


# ------------------------------------------------------------------ drawn cases

MOST_LOGITS = 2.2e8  # rows x heads x keys of a prefix case, whose plain form holds them in fp32 several times over


def _log_int(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _most(kind):
    costs = [work(case) for case in listed() if case["kind"] == kind]
    return {key: max(cost[key] for cost in costs) for key in ("bytes", "flops")}


def _draw_prefix(rng):
    kv = rng.choice((1, 2, 4, 8, 16))
    page = rng.choice((32, 64, 128))
    groups = rng.choice((1, 1, 2, _log_int(rng, 1, 16)))
    cut = rng.choice((0, 0, rng.randrange(page)))
    queries = rng.choice((1, 1, 1, 2, 4, 7))
    return {"kind": "prefix", "groups": groups, "batch": _log_int(rng, 1, 256 // groups),
            "shared": page * _log_int(rng, 1, 16000 // page), "cut": cut, "tail": cut + queries + _log_int(rng, 1, 2000),
            "queries": queries, "heads": kv * rng.choice((1, 2, 4, 7, 8)), "kv": kv,
            "dim": rng.choice((64, 128, 128, 256)), "page": page, "dtype": rng.choice(("bf16", "bf16", "f16", "f32"))}


def _draw_pages(rng):
    what = rng.choice(("step", "fork", "compact"))
    page = rng.choice((32, 64, 128))
    batch = _log_int(rng, 1, 128)
    tokens = max(batch, _log_int(rng, 1, 190000))
    case = {"kind": "pages", "what": what, "batch": batch, "tokens": tokens, "page": page, "kv": rng.choice((1, 2, 8)),
            "dim": rng.choice((64, 128, 256)), "layers": rng.choice((1, 2, 4)) if what != "step" else 0}
    needed = sum(-(-n // page) for n in _parts(tokens, batch))
    if what == "step":
        case.update(more=_log_int(rng, 1, 4 * page), window=rng.choice((0, _log_int(rng, 1, 4096))))
        needed += batch * (case["more"] // page + 2)
    if what == "fork":
        case["children"] = _log_int(rng, 1, 256)
        needed += case["children"]
    case["pages"] = int(needed * rng.uniform(1.0, 2.0)) + rng.randrange(40)
    return case


def _draw_score(rng):
    vocab = _log_int(rng, 2, 262144)
    return {"kind": "score", "rows": _log_int(rng, 1, 4096), "vocab": vocab,
            "top": min(vocab, rng.choice((0, 1, 5, 20, 64))), "dtype": rng.choice(("f32", "f16", "bf16")),
            "temperature": rng.choice((1.0, 0.7, 1.3))}


def _draw_rotate(rng):
    kv, dim = rng.choice((1, 2, 3, 4, 8, 16)), rng.choice((64, 128, 128, 256))
    tokens = _log_int(rng, 1, 8190)
    return {"kind": "rotate", "batch": min(tokens, _log_int(rng, 1, 64)), "tokens": tokens,
            "past": rng.choice((0, _log_int(rng, 1, 130000))), "heads": kv * rng.choice((1, 1, 2, 4, 7)), "kv": kv,
            "dim": dim, "rotary": rng.choice((dim, dim, dim // 2, dim // 4)), "norm": rng.random() < 0.6,
            "interleaved": rng.random() < 0.3, "base": rng.choice((10000.0, 500000.0)),
            "dtype": rng.choice(("bf16", "f16", "f32")), "fused": rng.random() < 0.5}


def draw(rng):
    kind = rng.choice(("prefix", "prefix", "pages", "score", "score", "rotate"))
    most = _most(kind)
    while True:
        case = {"prefix": _draw_prefix, "pages": _draw_pages, "score": _draw_score, "rotate": _draw_rotate}[kind](rng)
        cost = work(case)
        if any(cost[key] > limit for key, limit in most.items()):
            continue
        if kind == "prefix":
            rows = case["groups"] * case["batch"] * case["queries"]
            keys = case["shared"] + case["tail"]
            own_values = case["groups"] * case["batch"] * (case["tail"] + 2 * case["page"]) * case["kv"] * case["dim"]
            if rows * case["heads"] * keys > MOST_LOGITS or own_values > MOST_LOGITS:
                continue
        return case


# ------------------------------------------------------------------ sizes


def _parts(total, batch, spread=3.0):
    """`total` in `batch` parts of at least one, the largest up to `spread` times the smallest, in no order."""
    weights = [1.0 + (spread - 1.0) * ((7 * i + 3) % batch) / max(1, batch - 1) for i in range(batch)]
    parts = [max(1, int(total * w / sum(weights))) for w in weights]
    index = 0
    while sum(parts) != total:
        step = 1 if sum(parts) < total else -1
        if parts[index % batch] + step >= 1:
            parts[index % batch] += step
        index += 1
    return parts


def _tails(case):
    """Tokens behind the shared pages of every sequence of a prefix case: the new rows at least, the longest `tail`."""
    count = case["groups"] * case["batch"]
    least = case["queries"]
    tail = max(least, case["tail"] - case["cut"])
    return [max(least, tail - (tail // 2) * ((5 * i) % count) // count) for i in range(count)]


def _children(case):
    """Parents of a fork case's rows: the first rows take one parent each in turn, some parents have no child, and
    some rows stay empty."""
    batch = case["batch"]
    return [-1 if i % 29 == 28 else (i * 5 // 4) % batch for i in range(case["children"])]


def _copied(case):
    """Rows of a fork case that need a page of their own for the tokens of an unfinished page."""
    lengths, seen, copies = _parts(case["tokens"], case["batch"]), set(), 0
    for parent in _children(case):
        copies += parent >= 0 and parent in seen and lengths[parent] % case["page"] != 0
        seen.add(parent)
    return copies


def _page_bytes(case):
    return case["kv"] * (case["page"] // TILE) * 34 * case["dim"]


def work(case):
    if case["kind"] == "prefix":
        heads, kv, dim, queries = case["heads"], case["kv"], case["dim"], case["queries"]
        shared, tails = case["shared"] - case["cut"], [n + case["cut"] for n in _tails(case)]
        pairs = sum(queries * shared + sum(n - queries + 1 + i for i in range(queries)) for n in tails)
        keys = case["groups"] * shared + sum(tails)
        rows = len(tails) * queries
        return {"bytes": 2 * keys * kv * (dim * 17 // 32) + 2 * rows * heads * dim * DTYPES[case["dtype"]].itemsize,
                "flops": 4 * pairs * heads * dim}
    if case["kind"] == "pages":
        held = sum(-(-n // case["page"]) for n in _parts(case["tokens"], case["batch"]))
        if case["what"] == "step":  # two numbers per sequence for either call, the free pages' bits, the given pages
            given = case["batch"] * case["more"] // case["page"] + 1
            return {"bytes": 16 * case["batch"] + case["pages"] // 8 + 16 * given, "flops": case["pages"]}
        if case["what"] == "fork":  # old rows in, new rows out, their pages' counts, the copied pages
            lengths = _parts(case["tokens"], case["batch"])
            new = sum(-(-lengths[p] // case["page"]) for p in _children(case) if p >= 0)
            copied = 2 * _copied(case) * _page_bytes(case) * case["layers"]
            return {"bytes": 12 * held + 12 * new + copied, "flops": held + new}
        moved = held * max(0, case["pages"] - held) // case["pages"]  # pages lie at random
        return {"bytes": 8 * held + 4 * case["pages"] + 2 * moved * _page_bytes(case) * case["layers"],
                "flops": held + case["pages"]}
    if case["kind"] == "score":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * DTYPES[case["dtype"]].itemsize + case["rows"] * (16 + 12 * case["top"]),
                "flops": 6 * values}
    values = case["tokens"] * (case["heads"] + case["kv"]) * case["dim"]
    return {"bytes": 2 * values * DTYPES[case["dtype"]].itemsize, "flops": 8 * values}


# ------------------------------------------------------------------ inputs


def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + part)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)


def _rows(generator, shape):
    """N(0, 1) with 2% of the channels six times as large, as queries and keys have them."""
    x = torch.randn(shape, generator=generator, device="cuda")
    channels = torch.randperm(shape[-1], generator=generator, device="cuda")[:max(1, shape[-1] // 50)]
    x[..., channels] *= 6.0
    return x


def _filled_pages(generator, count, kv, page, dim):
    """Pages of normal values: codes as a normal number at half a scale step rounds to, and scales around 2^-1."""
    normal = torch.randn(1 << 17, generator=generator, device="cuda")
    middles = torch.tensor([(a + b) / 2 for a, b in zip(MAGNITUDES, MAGNITUDES[1:])], device="cuda")
    codes = (torch.bucketize(normal.abs() * 2, middles) + 8 * (normal < 0)).to(torch.uint8)
    codes = codes[0::2] + 16 * codes[1::2]
    pages = torch.empty((count, kv, page // TILE, 34 * dim), dtype=torch.uint8, device="cuda")
    for part in pages.split(max(1, (1 << 27) // pages[0].numel())):
        index = torch.randint(0, 1 << 16, (*part.shape[:3], 32 * dim), generator=generator, device="cuda")
        part[..., :32 * dim] = codes[index]
        part[..., 32 * dim:] = torch.randint(125, 128, (*part.shape[:3], 2 * dim), generator=generator, device="cuda",
                                             dtype=torch.uint8)
    return pages


def _prepare_prefix(case, seed):
    generator = _generator(seed, 1)
    page, groups, batch, queries = case["page"], case["groups"], case["batch"], case["queries"]
    tails, shared = _tails(case), case["shared"]
    width = shared // page + -(-max(tails) // page) + 1
    own_pages = [-(-n // page) for n in tails]
    total = groups * (shared // page) + sum(own_pages) + 3
    order = torch.randperm(total, generator=generator, device="cuda").to(torch.int32)
    table = torch.full((groups * batch, width), -1, dtype=torch.int32, device="cuda")
    start = 0
    for group in range(groups):
        table[group * batch:(group + 1) * batch, :shared // page] = order[start:start + shared // page]
        start += shared // page
    for row, count in enumerate(own_pages):
        table[row, shared // page:shared // page + count] = order[start:start + count]
        start += count
    rows = groups * batch * queries
    return {"kind": "prefix", "dtype": DTYPES[case["dtype"]], "table": table,
            "pages": _filled_pages(generator, total, case["kv"], page, case["dim"]),
            "q": _rows(generator, (rows, case["heads"], case["dim"])).to(DTYPES[case["dtype"]]),
            "lengths": _ints([shared + n for n in tails]), "groups": _ints([batch * g for g in range(groups + 1)]),
            "prefix": _ints([shared - case["cut"]] * groups), "queries": queries, "batch": batch,
            "offsets": None if queries == 1 else _ints([queries * b for b in range(groups * batch + 1)]),
            "most_prefix": shared - case["cut"], "longest": shared + max(tails)}


def _free_words(refs):
    bits = torch.nn.functional.pad((refs == 0).long(), (0, -refs.shape[0] % 32)).view(-1, 32)
    words = (bits << torch.arange(32, device="cuda")).sum(1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _prepare_pages(case, seed):
    generator = _generator(seed, 2)
    page, total = case["page"], case["pages"]
    lengths = _parts(case["tokens"], case["batch"])
    if seed % 2:  # another order of the lengths, and other fill levels of the last pages
        lengths = lengths[::-1]
    needed = [-(-n // page) for n in lengths]
    more = case.get("more", 0)
    width = max(needed) + more // page + 2
    order = torch.randperm(total, generator=generator, device="cuda").to(torch.int32)
    table = torch.full((len(needed), width), -1, dtype=torch.int32, device="cuda")
    start = 0
    for row, count in enumerate(needed):
        table[row, :count] = order[start:start + count]
        start += count
    refs = torch.zeros(total, dtype=torch.int32, device="cuda")
    refs[order[:start].long()] = 1
    # the table, the counts and the free pages' bits side by side: a pass starts from `saved`
    saved = torch.cat((table.flatten(), refs, _free_words(refs)))
    live = saved.clone()
    words = (total + 31) // 32
    cut = table.numel()
    state = {"kind": "pages", "what": case["what"], "saved": saved, "live": live, "page": page,
             "table": live[:cut].view(table.shape), "refs": live[cut:cut + total],
             "free": live[cut + total:cut + total + words], "lengths": _ints(lengths),
             "layers": [_filled_pages(generator, total, case["kv"], page, case["dim"]) for _ in range(case["layers"])]}
    if case["what"] == "step":
        window = case["window"]
        state.update(counts=_ints([more] * len(lengths)), first=_ints([0] * len(lengths)),
                     last=_ints([max(0, n + more - window) // page if window else 0 for n in lengths]))
    if case["what"] == "fork":
        state["parents"] = _ints(_children(case))
    return state


def _prepare_score(case, seed):
    generator = _generator(seed, 3)
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty((rows, vocab), dtype=DTYPES[case["dtype"]], device="cuda")
    for part in logits.split(max(1, (1 << 26) // vocab)):
        part.copy_(torch.randn(part.shape, generator=generator, device="cuda") * 2.5)
    likely = torch.randint(0, vocab, (rows, 8), generator=generator, device="cuda")
    peaks = (torch.randn((rows, 8), generator=generator, device="cuda") * 2 + 9).to(logits.dtype)
    for j in range(8):  # one after another: a token may be drawn twice
        logits.scatter_(1, likely[:, j:j + 1], peaks[:, j:j + 1])
    random = torch.randint(0, vocab, (rows,), generator=generator, device="cuda")
    tokens = torch.where(torch.arange(rows, device="cuda") % 4 == 3, random, likely[:, 0])
    return {"kind": "score", "logits": logits, "tokens": tokens, "top": case["top"], "temperature": case["temperature"]}


def _prepare_rotate(case, seed):
    generator = _generator(seed, 4)
    rows, heads, kv, dim = case["tokens"], case["heads"], case["kv"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    if case["fused"]:  # q, k and v side by side, as one projection leaves them
        fused = _rows(generator, (rows, heads + 2 * kv, dim)).to(dtype)
        q, k = fused[:, :heads], fused[:, heads:heads + kv]
    else:
        q, k = (_rows(generator, (rows, n, dim)).to(dtype) for n in (heads, kv))
    counts = _parts(rows, case["batch"])
    past = [case["past"] * (b + 1) // case["batch"] for b in range(case["batch"])]
    half = torch.arange(case["rotary"] // 2, dtype=torch.float64, device="cuda")
    norms = [None, None]
    if case["norm"]:
        norms = [1.0 + 0.2 * torch.randn(dim, generator=generator, device="cuda") for _ in range(2)]
    return {"kind": "rotate", "q": q, "k": k, "past": _ints(past), "offsets": _offsets(counts), "dtype": dtype,
            "frequencies": (case["base"] ** (-2.0 * half / case["rotary"])).float(), "q_norm": norms[0],
            "k_norm": norms[1], "eps": 1e-6, "interleaved": case["interleaved"]}


def prepare(case, seed):
    return {"prefix": _prepare_prefix, "pages": _prepare_pages, "score": _prepare_score,
            "rotate": _prepare_rotate}[case["kind"]](case, seed)


# ------------------------------------------------------------------ plain forms: prefix


def _tile_bytes(dim):
    """Byte of a tile that holds dims 2 i, 2 i + 1 of token t, and the scale byte of 32 dims: of K and of V,
    [32, dim / 2] and [32, dim / 32]."""
    t, byte, group = (torch.arange(n, device="cuda") for n in (TILE, dim // 2, dim // 32))
    t, width = t[:, None], dim // 32
    e, b = t // 16 * 4 + t % 4, t % 16 // 4
    per = 16 // width
    k = t * (dim // 2) + byte
    v = 16 * dim + e // per * 1024 + (b * 16 + byte // width) * 16 + e % per * width + byte % width
    return k, v, 32 * dim + group * 32 + t % 16 * 2 + t // 16, 33 * dim + group * 32 + b * 8 + e


def _values(tiles, codes, scales):
    """fp32 values [..., 32, dim] of tiles [..., 34 * dim], from the places of their codes and scales."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device="cuda")
    packed = tiles[..., codes]
    nibbles = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    return table[nibbles.int()] * torch.exp2(tiles[..., scales].float() - 127).repeat_interleave(32, -1)


def _gathered(pages, entries):
    """K and V [..., kv, tokens, dim] of table entries [..., pages]; entries without a page give those of page 0."""
    dim = pages.shape[-1] // 34
    tiles = pages[entries.clamp_min(0).long()].transpose(-3, -4)  # [..., kv, pages, tiles, bytes]
    k, v, k_scale, v_scale = _tile_bytes(dim)
    return (_values(tiles, k, k_scale).flatten(-4, -2), _values(tiles, v, v_scale).flatten(-4, -2))


def _prefix(s):
    """The shared keys once for all rows of a group, the rest for each sequence, one softmax over both."""
    q, pages, table, batch, n = s["q"], s["pages"], s["table"], s["batch"], s["queries"]
    heads, dim = q.shape[1:]
    kv = pages.shape[1]
    page = pages.shape[2] * TILE
    prefix, longest = s["most_prefix"], s["longest"]
    scale = dim ** -0.5
    out = torch.empty_like(q)
    for group in range(table.shape[0] // batch):
        members = slice(group * batch, (group + 1) * batch)
        rows = slice(group * batch * n, (group + 1) * batch * n)
        k, v = (x[:, :prefix] for x in _gathered(pages, table[members][0, :-(-prefix // page)]))
        first = prefix // page
        entries = table[members][:, first:-(-longest // page)]
        k_own, v_own = (x[:, :, prefix - first * page:] for x in _gathered(pages, entries))
        own_keys = k_own.shape[2]
        grouped = q[rows].float().view(batch, n, kv, heads // kv, dim).permute(2, 0, 3, 1, 4)  # [kv, B, g, n, D]
        shared = torch.matmul(grouped.reshape(kv, -1, dim), k.transpose(1, 2).contiguous())
        behind = torch.matmul(grouped.transpose(0, 1).reshape(batch, kv, -1, dim), k_own.transpose(-1, -2).contiguous())
        position = s["lengths"][members].long()[:, None] - n + torch.arange(n, device="cuda")
        seen = prefix + torch.arange(own_keys, device="cuda") <= position[:, :, None]  # [B, n, keys]
        behind = behind.view(batch, kv, heads // kv, n, own_keys).masked_fill(~seen[:, None, None], -math.inf)
        scores = torch.cat((shared.view(kv, batch, -1, n, prefix).transpose(0, 1), behind), -1).mul_(scale)
        weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        total = weights.sum(-1)
        of_shared = weights[..., :prefix].transpose(0, 1).reshape(kv, -1, prefix)
        of_own = weights[..., prefix:].reshape(batch, kv, -1, own_keys)
        result = torch.matmul(of_own, v_own).view(batch, kv, -1, n, dim)
        result += torch.matmul(of_shared, v).view(kv, batch, -1, n, dim).transpose(0, 1)
        result /= total[..., None]
        out[rows] = result.permute(0, 3, 1, 2, 4).reshape(batch * n, heads, dim).to(out.dtype)
    return out


# ------------------------------------------------------------------ plain forms: pages


def _free_order(refs):
    """The pages, free ones first and by number, and how many are free."""
    free = refs == 0
    return torch.sort((~free).byte(), stable=True).indices, free.sum()


def _reserve(s):
    table, refs, page = s["table"], s["refs"], s["page"]
    width = table.shape[1]
    lengths = s["lengths"].long().clamp_min(0)
    first = (lengths + page - 1) // page
    last = (lengths + s["counts"].clamp_min(0) + page - 1) // page
    slot = torch.arange(width, device="cuda")
    valid = (table >= 0) & (table < refs.shape[0])
    need = (slot >= first[:, None]) & (slot < last[:, None]) & ~valid
    order, available = _free_order(refs)
    rank = need.flatten().cumsum(0).view_as(table) - 1
    got = need & (rank < available)
    chosen = order[rank.clamp(0, refs.shape[0] - 1)]
    outside = (last.clamp_min(width) - first.clamp_min(width)).sum()
    table.copy_(torch.where(got, chosen.to(torch.int32), table))
    refs.scatter_add_(0, chosen.flatten(), got.flatten().to(torch.int32))
    s["free"].copy_(_free_words(refs))
    return ((need & ~got).sum() + outside).to(torch.int32).view(1)


def _release(s):
    table, refs = s["table"], s["refs"]
    slot = torch.arange(table.shape[1], device="cuda")
    mask = (slot >= s["first"][:, None]) & (slot < s["last"][:, None]) & (table >= 0) & (table < refs.shape[0])
    refs.scatter_add_(0, table.clamp(0, refs.shape[0] - 1).long().flatten(), -mask.flatten().to(torch.int32))
    table.masked_fill_(mask, -1)
    s["free"].copy_(_free_words(refs))


def _fork(s):
    table, refs, page, parents = s["table"], s["refs"], s["page"], s["parents"].long()
    batch, width = table.shape
    count = parents.shape[0]
    there = (parents >= 0) & (parents < batch)
    parent = parents.clamp(0, batch - 1)
    lengths = torch.where(there, s["lengths"].long()[parent].clamp_min(0), 0)
    whole = lengths // page
    child = torch.arange(count, device="cuda")
    first = torch.full((batch,), count, device="cuda")
    first.scatter_reduce_(0, parent, torch.where(there, child, count), "amin")
    heir = there & (first[parent] == child)
    rows = table[parent]
    slot = torch.arange(width, device="cuda")
    new = torch.where(there[:, None] & (heir[:, None] | (slot < whole[:, None])), rows, -1)
    source = rows.gather(1, whole.clamp_max(width - 1)[:, None])[:, 0]
    wants = there & ~heir & (lengths % page != 0) & (whole < width) & (source >= 0) & (source < refs.shape[0])
    order, available = _free_order(refs)
    rank = wants.cumsum(0) - 1
    got = wants & (rank < available)
    target = order[rank.clamp(0, refs.shape[0] - 1)].to(torch.int32)
    place = whole.clamp_max(width - 1)[:, None]
    new.scatter_(1, place, torch.where(got, target, new.gather(1, place)[:, 0])[:, None])
    copies = torch.full((count + 1, 2), -1, dtype=torch.int32, device="cuda")
    copies[torch.where(got, rank, count)] = torch.where(got[:, None], torch.stack((source, target), 1), -1)
    lengths = torch.where(wants & ~got, whole * page, lengths)
    for rows, step in ((new, 1), (table, -1)):
        valid = (rows >= 0) & (rows < refs.shape[0])
        refs.scatter_add_(0, rows.clamp(0, refs.shape[0] - 1).long().flatten(), valid.flatten().to(torch.int32) * step)
    s["free"].copy_(_free_words(refs))
    return new, lengths.to(torch.int32), copies[:count], (wants & ~got).sum().to(torch.int32).view(1)


def _compact(s):
    table, refs = s["table"], s["refs"]
    total = refs.shape[0]
    held = refs > 0
    live = held.sum()
    number = torch.arange(total, device="cuda")
    hole, mover = ~held & (number < live), held & (number >= live)
    most = (total + 1) // 2
    target = torch.full((most + 1,), -1, device="cuda")
    target[torch.where(hole, hole.cumsum(0) - 1, most)] = torch.where(hole, number, -1)
    rank = torch.where(mover, mover.cumsum(0) - 1, most)
    copies = torch.full((most + 1, 2), -1, dtype=torch.int32, device="cuda")
    copies[rank] = torch.where(mover[:, None], torch.stack((number, target[rank]), 1), -1).to(torch.int32)
    moved = torch.where(mover, target[rank], number)
    valid = (table >= 0) & (table < total)
    table.copy_(torch.where(valid, moved[table.clamp(0, total - 1).long()].to(torch.int32), table))
    refs.copy_(torch.zeros_like(refs).scatter_add_(0, moved, torch.where(held, refs, 0)))
    s["free"].copy_(_free_words(refs))
    return copies[:total // 2], live.to(torch.int32).view(1)


def _copy(pages, copies):
    """Rows without a copy take a page onto itself: the first copy's source."""
    source = torch.where(copies[:, 0] >= 0, copies[:, 0], copies[0, 0].clamp_min(0)).long()
    target = torch.where(copies[:, 0] >= 0, copies[:, 1], copies[0, 0].clamp_min(0)).long()
    pages[target] = pages[source]


def _pages(s):
    s["live"].copy_(s["saved"])
    if s["what"] == "step":
        short = _reserve(s)
        _release(s)
        return s["table"], s["refs"], s["free"], short
    if s["what"] == "fork":
        table, lengths, copies, short = _fork(s)
        for pages in s["layers"]:
            _copy(pages, copies)
        return table, lengths, s["refs"], s["free"], short, s["layers"]
    copies, live = _compact(s)
    for pages in s["layers"]:
        _copy(pages, copies)
    return s["table"], s["refs"], s["free"], live, s["layers"]


# ------------------------------------------------------------------ plain forms: score and rotate


def _order_keys(logits):
    """A 64-bit number per logit: larger logits have larger ones, and of equal logits the one of the lower index."""
    bits = (logits.float() + 0.0).view(torch.int32).long()
    ordered = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    return (ordered << 32) - torch.arange(logits.shape[1], device="cuda")


def _score(s):
    logits, tokens, top = s["logits"], s["tokens"], s["top"]
    x = logits.float() / s["temperature"]
    most = x.amax(1, keepdim=True)
    x = x - most
    weights = x.exp()
    total = weights.sum(1)
    log_total = total.log()
    entropy = log_total - (x * weights).sum(1) / total
    chosen = x.gather(1, tokens[:, None])[:, 0] - log_total
    if top == 0:
        best = torch.empty((logits.shape[0], 0), dtype=torch.int64, device="cuda")
    else:
        best = torch.topk(_order_keys(logits), top, dim=1).indices
    return chosen, entropy, x.gather(1, best) - log_total[:, None], best


def _positions(s, rows):
    row = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    return s["past"].long()[sequence] + row - s["offsets"].long()[sequence]


def _rotate(s):
    # angles of far positions lose their fraction in 32 bits
    angle = _positions(s, s["q"].shape[0]).double()[:, None, None] * s["frequencies"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    half = cos.shape[-1]
    results = []
    for x, weight in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * weight
        turned = x[..., :2 * half]
        if s["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            pair = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = turned[..., :half], turned[..., half:]
            pair = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        results.append(torch.cat((pair, x[..., 2 * half:]), -1).to(s["dtype"]))
    return tuple(results)


# ------------------------------------------------------------------ one pass


def run(state):
    if own:
        return _run_own(state)
    return {"prefix": _prefix, "pages": _pages, "score": _score, "rotate": _rotate}[state["kind"]](state)


def _modules(s):
    modules = s.get("modules")
    if modules is None:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ivonar-inference_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from ivonar_amd import attention, paging, sampling

        modules = s["modules"] = (attention, paging, sampling)
        if s["kind"] == "pages":
            s["pool"] = paging.PagePool(s["refs"], s["free"], s["page"])
    return modules


def _run_own(s):
    attention, paging, sampling = _modules(s)
    if s["kind"] == "prefix":
        return attention.prefix_attention(s["q"], s["pages"], s["table"], s["lengths"], s["groups"], s["prefix"],
                                          s["offsets"], max_length=s["longest"], max_prefix=s["most_prefix"])
    if s["kind"] == "score":
        return tuple(sampling.log_probabilities(s["logits"], s["tokens"], s["top"], s["temperature"]))
    if s["kind"] == "rotate":
        return attention.rotate(s["q"], s["k"], s["past"], s["frequencies"], s["offsets"], s["q_norm"], s["k_norm"],
                                s["eps"], s["interleaved"])
    pool, table = s["pool"], s["table"]
    s["live"].copy_(s["saved"])
    if s["what"] == "step":
        short = paging.reserve(pool, table, s["lengths"], s["counts"])
        paging.release(pool, table, s["first"], s["last"])
        return table, pool.refs, pool.free, short
    if s["what"] == "fork":
        new, lengths, copies, short = paging.fork(pool, table, s["lengths"], s["parents"])
        for pages in s["layers"]:
            paging.copy(pages, copies)
        return new, lengths, pool.refs, pool.free, short, s["layers"]
    copies, live = paging.compact(pool, table)
    for pages in s["layers"]:
        paging.copy(pages, copies)
    return table, pool.refs, pool.free, live, s["layers"]


# ------------------------------------------------------------------ answers in 64 bits


def _tile_values(tiles, dim):
    """K and V [n, 32, dim] in 64 bits of tiles uint8 [n, 34 * dim], by the order in which a tile's bytes lie."""
    def four(code):
        low = code & 7
        value = torch.where(low < 2, low * 0.5, (1 + (low & 1) * 0.5) * 2.0 ** ((low >> 1) - 1))
        return torch.where(code >= 8, -value, value)

    def two(byte):
        return torch.stack((four(byte & 15), four(byte >> 4)), -1).double()

    tiles = tiles.long()
    count, width = tiles.shape[0], dim // 32
    k = two(tiles[:, :16 * dim]).reshape(count, 32, dim)
    v = two(tiles[:, 16 * dim:32 * dim]).reshape(count, width // 2, 4, 16, 16 // width, 2 * width)
    v = v.permute(0, 1, 4, 2, 3, 5).reshape(count, 2, 4, 4, dim).transpose(2, 3).reshape(count, 32, dim)
    k_scale = tiles[:, 32 * dim:33 * dim].reshape(count, width, 16, 2).permute(0, 3, 2, 1).reshape(count, 32, width)
    v_scale = tiles[:, 33 * dim:].reshape(count, width, 4, 2, 4).permute(0, 3, 2, 4, 1).reshape(count, 32, width)
    return tuple((x.unflatten(-1, (-1, 32)) * 2.0 ** (e - 127).double()[..., None]).flatten(-2)
                 for x, e in ((k, k_scale), (v, v_scale)))


def _exact_prefix(s):
    """Every sequence by itself over all of its tokens."""
    q, pages, n = s["q"].double(), s["pages"], s["queries"]
    kv, tiles, size = pages.shape[1:]
    dim, heads = size // 34, q.shape[1]
    out = torch.empty_like(q)
    for b, length in enumerate(s["lengths"].tolist()):
        entries = s["table"][b, :-(-length // (tiles * TILE))].long()
        chosen = pages[entries].transpose(0, 1).reshape(-1, size)
        k, v = (x.reshape(kv, -1, dim)[:, :length] for x in _tile_values(chosen, dim))
        rows = q[b * n:(b + 1) * n].transpose(0, 1).reshape(kv, -1, dim)  # [kv, group * n, dim]
        scores = torch.matmul(rows, k.transpose(1, 2)) / math.sqrt(dim)
        hidden = torch.arange(length, device="cuda") > (length - n + torch.arange(n, device="cuda"))[:, None]
        scores.view(kv, -1, n, length).masked_fill_(hidden, -math.inf)
        result = torch.matmul(torch.softmax(scores, -1), v)
        out[b * n:(b + 1) * n] = result.reshape(heads, n, dim).transpose(0, 1)
    return out


def _exact_score(s):
    logits, top = s["logits"], s["top"]
    parts = []
    for x, token in zip(logits.split(256), s["tokens"].split(256)):
        logs = torch.log_softmax(x.double() / s["temperature"], 1)
        entropy = -(logs.exp() * logs).sum(1)
        best = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
        parts.append((logs.gather(1, token[:, None])[:, 0], entropy, logs.gather(1, best), best))
    return tuple(torch.cat(side) for side in zip(*parts))


def _exact_rotate(s):
    """Pairs of dims as complex numbers, turned by e^(i position frequency)."""
    position = _positions(s, s["q"].shape[0]).double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), position[:, None] * s["frequencies"].double())
    half = turn.shape[1]
    results = []
    for x, weight in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        x = x.double()
        if weight is not None:
            x = weight.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + s["eps"])
        out = x.clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["interleaved"] else (
            slice(0, half), slice(half, 2 * half))
        turned = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn[:, None]
        out[..., first], out[..., second] = turned.real, turned.imag
        results.append(out)
    return tuple(results)


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers and bytes
    state = prepare(case, seed)
    return {"prefix": _exact_prefix, "score": _exact_score, "rotate": _exact_rotate}[case["kind"]](state)
