"""Operators of a serving cache: keys and values in pages of 4-bit numbers.

A page holds ``page_size`` keys and values of every KV head as E2M1 numbers in
blocks of 32 that share a power of two.  Three operators use such caches: storing
new keys and values, with what the cache then holds read back (``store``), the
attention of new tokens over the pages of their sequences (``attention``), and the
pages themselves, continued by other sequences (``fork``) or moved to the front
of the cache (``compact``).  ``listed`` holds one size of each use, ``draw`` the
ranges.  ``run`` computes the definitions in elementary operations, or, with
``own``, makes the calls that a user of this package makes.
"""

import math
import os
import sys

import torch

own = False

BLOCK = 32          # elements that share an exponent
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # of the codes 0..7; bit 3 is the sign
LEAST, MOST = 27, 252  # the exponent's byte: 2^-100 to 2^125


def listed():
    return [
        # A decoding step's keys and values: one token of 64 sequences.
        {"name": "store_decode", "op": "store", "dtype": "bf16", "batch": 64, "tokens": 1, "keys": 2048, "hkv": 8,
         "hd": 128, "page": 64},
        # A long prompt, and what the cache holds of it for the prompt's own attention.
        {"name": "store_prefill", "op": "store", "dtype": "bf16", "batch": 1, "tokens": 16001, "keys": 16001, "hkv": 8,
         "hd": 128, "page": 64},
        # A padded FP16 batch of prompts of different lengths, heads of 64, small pages.
        {"name": "store_ragged", "op": "store", "dtype": "f16", "batch": 7, "tokens": 1000, "keys": 1000, "hkv": 4,
         "hd": 64, "page": 16},
        # Decoding with few short sequences: launches and latency.
        {"name": "decode_small", "op": "attention", "dtype": "bf16", "batch": 8, "tokens": 1, "keys": 1200, "hq": 32,
         "hkv": 8, "hd": 128, "page": 64, "softcap": 0.0},
        # A full server's decoding step, lengths from a single key to the cache's end.
        {"name": "decode_batch", "op": "attention", "dtype": "bf16", "batch": 64, "tokens": 1, "keys": 16384, "hq": 32,
         "hkv": 8, "hd": 128, "page": 64, "softcap": 0.0},
        # Two very long sequences: few rows, one long axis.
        {"name": "decode_long", "op": "attention", "dtype": "bf16", "batch": 2, "tokens": 1, "keys": 131072, "hq": 32,
         "hkv": 8, "hd": 128, "page": 32, "softcap": 0.0},
        # Softcapped scores, ungrouped heads of 64, odd lengths, FP16, the smallest pages.
        {"name": "decode_softcap", "op": "attention", "dtype": "f16", "batch": 33, "tokens": 1, "keys": 8191, "hq": 16,
         "hkv": 16, "hd": 64, "page": 16, "softcap": 30.0},
        # Five proposed tokens of each sequence are verified at once.
        {"name": "verify_tokens", "op": "attention", "dtype": "bf16", "batch": 32, "tokens": 5, "keys": 4100, "hq": 32,
         "hkv": 4, "hd": 128, "page": 64, "softcap": 0.0},
        # A piece of each prompt behind what the cache holds of it.
        {"name": "extend", "op": "attention", "dtype": "bf16", "batch": 4, "tokens": 512, "keys": 8700, "hq": 32,
         "hkv": 8, "hd": 128, "page": 64, "softcap": 0.0},
        # A step of a beam search: 16 beams, two of each surviving one.
        {"name": "fork_beams", "op": "fork", "layers": 4, "pages": 512, "rows": 16, "fanout": 2, "entries": 24,
         "page": 64, "hkv": 8, "hd": 128},
        # Four answers to each of 64 prompts.
        {"name": "fork_samples", "op": "fork", "layers": 8, "pages": 4096, "rows": 256, "fanout": 4, "entries": 48,
         "page": 64, "hkv": 8, "hd": 128},
        # A cache that other sequences have left in holes moves to its front.
        {"name": "compact", "op": "compact", "layers": 8, "pages": 4096, "used": 2048, "entries": 64, "page": 64,
         "hkv": 8, "hd": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attention", "attention", "attention", "fork", "compact"])
    page, hd, hkv = rng.choice([16, 32, 64, 128]), rng.choice([64, 128]), rng.choice([1, 2, 4, 8, 16])
    case = {"op": op, "page": page, "hd": hd, "hkv": hkv}
    if op in ("fork", "compact"):
        layers = rng.choice([1, 2, 4, 8])
        most = min(16384, 8 * 4096 * 64 * 8 * 128 // (layers * page * hkv * hd))
        pages = _log(rng, 64, most)
        if op == "compact":
            return {**case, "layers": layers, "pages": pages, "used": rng.randint(pages // 4, pages * 3 // 4),
                    "entries": _log(rng, 4, 256)}
        fanout, rows = rng.choice([1, 2, 3, 4]), _log(rng, 4, 256)
        rows = max(rows // fanout, 1) * fanout
        entries = _log(rng, 2, 128)
        need = rows // fanout * entries + 2 * rows  # the survivors' pages, copies and new ones
        return {**case, "layers": layers, "pages": max(pages, need), "rows": rows, "fanout": fanout,
                "entries": entries} if need <= most else draw(rng)
    case["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    if op == "store":
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, 16000)
        batch = _log(rng, 1, max(1, min(256, 16001 * 8 * 128 // (tokens * hkv * hd))))
        return {**case, "batch": batch, "tokens": tokens, "keys": tokens + _log(rng, 1, 4096) - 1}
    hq = hkv * rng.choice([1, 2, 4, 8])
    hq = min(hq, max(hkv, 64 // hkv * hkv))
    keys = _log(rng, 16, 131072)
    # at most the keys, and the rows times keys, of the largest listed cases
    most = max(1, 64 * 16384 * 8 * 128 // (keys * hkv * hd))
    rows = max(1, min(2048, 4 * 512 * 8700 * 32 * 128 // (keys * hq * hd)))
    tokens = 1 if rng.random() < 0.6 else _log(rng, 2, max(2, min(512, rows)))
    batch = _log(rng, 1, max(1, min(256, most, rows // tokens)))
    return {**case, "batch": batch, "tokens": tokens, "keys": max(keys, tokens), "hq": hq,
            "softcap": rng.choice([0.0, 0.0, 30.0, 50.0])}


def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.bfloat16


def _lens(case):
    """Valid keys of each sequence: from the new tokens alone (a padded batch's
    prompts: from half of them) to all."""
    b, t, n = case["batch"], case["tokens"], case["keys"]
    if b == 1:
        return [n]
    least = (t + 1) // 2 if case["op"] == "store" else t
    return [least + (n - least) * i // (b - 1) for i in range(b)]


def _page_bytes(case):
    """Of one KV head's keys or values: the codes and the blocks' exponents."""
    return case["page"] * (case["hd"] // 2 + case["hd"] // BLOCK)


def _random_cache(case, pages, g):
    """[pages, 2, hkv, bytes]: any codes, exponents of keys and values about 1."""
    codes = case["page"] * case["hd"] // 2
    cache = torch.randint(0, 256, (pages, 2, case["hkv"], _page_bytes(case)), generator=g, device="cuda",
                          dtype=torch.uint8)
    cache[..., codes:] = cache[..., codes:] % 3 + 124
    return cache


def _inputs(case, seed):
    """The operands, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    page = case["page"]
    if case["op"] in ("fork", "compact"):
        pages, entries = case["pages"], case["entries"]
        x = {"caches": [_random_cache(case, pages, g) for _ in range(case["layers"])]}
        order = torch.randperm(pages, generator=h).to(torch.int32)
        if case["op"] == "compact":
            used, moved = case["used"], _moved(case)
            low = torch.randperm(used, generator=h)[: used - moved]
            high = used + torch.randperm(pages - used, generator=h)[:moved]
            ids = torch.cat([low, high])[torch.randperm(used, generator=h)].to(torch.int32)
            table = torch.full((-(-used // entries) * entries,), -1, dtype=torch.int32)
            table[:used] = ids
            return {**x, "table": table.view(-1, entries).cuda()}
        rows, alive = case["rows"], case["rows"] // case["fanout"]
        lens = torch.randint(1, entries * page, (rows,), generator=h)
        lens += (lens % page == 0).long()  # the last page is never full: each further row copies it
        table = torch.full((rows, entries + 1), -1, dtype=torch.int32)
        parents = torch.randperm(rows, generator=h)[:alive]  # the others end
        at = 0
        for row in range(rows):
            n = -(-int(lens[row]) // page)
            if row in parents or at + n <= pages - (alive * entries + 2 * rows):
                table[row, :n] = order[at: at + n]
                at += n
            else:
                lens[row] = 0
        parents = parents.repeat(case["fanout"])[torch.randperm(rows, generator=h)]
        return {**x, "table": table.cuda(), "lens": lens.to(torch.int32).cuda(),
                "parents": parents.to(torch.int32).cuda()}
    dt, b, t, hkv, d = _dtype(case), case["batch"], case["tokens"], case["hkv"], case["hd"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt).mul_(scale)

    lens = torch.tensor(_lens(case), dtype=torch.int32)[torch.randperm(b, generator=h)]
    entries = -(-case["keys"] // page)
    counts = (lens.long() + page - 1) // page
    table = torch.full((b, entries), -1, dtype=torch.int32)
    order = torch.randperm(int(counts.sum()) + 8, generator=h).to(torch.int32)  # pages in any order, some free
    held = torch.arange(entries)[None] < counts[:, None]
    table[held] = order[: int(counts.sum())]
    x = {"table": table.cuda(), "lens": lens.cuda(), "cache": _random_cache(case, order.numel(), g)}
    if case["op"] == "store":
        # views of the packed projection; a few channels are far larger than the others
        qkv = normal(b, t, 3 * hkv * d)
        qkv[..., :: 37] *= 12
        x["k"], x["v"] = (qkv[..., i * hkv * d: (i + 1) * hkv * d].unflatten(-1, (hkv, d)) for i in (1, 2))
    else:
        x["q"] = normal(b, t, case["hq"], d, scale=8.0 if case["softcap"] else 1.0)  # up to a softcap's bend
    return x


def _moved(case):
    """Pages behind the first ``used`` that are in use, where any page may be."""
    return case["used"] * (case["pages"] - case["used"]) // case["pages"]


def prepare(case, seed):
    return {"case": dict(case), **_inputs(case, seed)}


# ---- the framework's calls ----------------------------------------------------

def _framework():
    path = os.path.join(os.getcwd(), "fast-polynomial-transcendentals_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sfu_repro import fa4_runtime, paged_cache
    return fa4_runtime, paged_cache


def _call(state):
    case = state["case"]
    fa4_runtime, paged_cache = _framework()
    if case["op"] == "attention":
        return fa4_runtime.flash_attn_paged_fp4(state["q"], state["cache"], state["table"], state["lens"],
                                                softcap=case["softcap"])
    if case["op"] == "store":
        paged_cache.store_fp4(state["cache"], state["k"], state["v"], state["table"], state["lens"])
        return paged_cache.load_fp4(state["cache"], state["table"], state["lens"], case["tokens"], case["hd"],
                                    dtype=_dtype(case))
    if case["op"] == "fork":
        return [*paged_cache.fork_pages(state["caches"], state["table"], state["lens"], state["parents"], tokens=1,
                                        page_size=case["page"]), *state["caches"]]
    return [*paged_cache.compact_pages(state["caches"], state["table"]), *state["caches"]]


# ---- the same in elementary operations, in 32 bits ------------------------------

def _halves(case, cache):
    """The codes [.., page, hd / 2] and the exponents' bytes [.., page, hd / 32]."""
    n = case["page"] * case["hd"] // 2
    return cache[..., :n].unflatten(-1, (case["page"], -1)), cache[..., n:].unflatten(-1, (case["page"], -1))


def _quantise(x):
    """Codes, two to a byte, and the blocks' bytes of [.., hd] values.  The power of
    two puts the block's largest value at 3.5 to 7 (to 6 after rounding)."""
    f = x.float().unflatten(-1, (-1, BLOCK))
    top = f.abs().amax(-1)
    byte = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(LEAST, MOST)
    y = f * ((254 - byte) << 23).view(torch.float32)[..., None]  # by 2^(127 - byte), exact
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5).int()) + 8 * (y < 0).int()
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), byte.to(torch.uint8)


def _values(codes, bytes_):
    """The float32 numbers that codes and exponents stand for."""
    lut = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    pairs = torch.stack([lut.repeat(16), lut.repeat_interleave(16)], -1)  # of a byte
    v = pairs.index_select(0, codes.reshape(-1).int()).view(*codes.shape[:-1], -1, BLOCK)
    return (v * torch.exp2(bytes_.float() - 127)[..., None]).flatten(-2)


def _token_rows(state):
    """Page, row in it and validity [batch, tokens] of each new token."""
    case, t = state["case"], state["case"]["tokens"]
    pos = state["lens"].long()[:, None] - t + torch.arange(t, device="cuda")
    entry = (pos // case["page"]).clamp(0, state["table"].shape[1] - 1)
    page = state["table"].long().gather(1, entry)
    return page, pos % case["page"], (pos >= 0) & (pos < state["table"].shape[1] * case["page"]) & (page >= 0)


def _plain_store(state):
    case = state["case"]
    page, row, valid = _token_rows(state)
    codes, bytes_ = _halves(case, state["cache"])
    p, r = page[valid], row[valid]
    for i, name in enumerate(("k", "v")):
        c, e = _quantise(state[name])
        codes[p, i, :, r], bytes_[p, i, :, r] = c[valid], e[valid]
    out = []
    for i in range(2):
        v = _values(codes[page.clamp_min(0), i, :, row], bytes_[page.clamp_min(0), i, :, row])
        v = v * valid[..., None, None]
        out.append((v.clamp(-65504, 65504) if case["dtype"] == "f16" else v).to(_dtype(case)))
    return out


def _plain_attention(state):
    """Token t of sequence b sees the keys 0 .. lens[b] - T + t."""
    case = state["case"]
    b, t, hq, hkv, d = case["batch"], case["tokens"], case["hq"], case["hkv"], case["hd"]
    group, n = hq // hkv, state["table"].shape[1] * case["page"]
    pages = state["cache"].index_select(0, state["table"].clamp_min(0).reshape(-1)).view(b, -1, 2, hkv, _page_bytes(case))
    k, v = (_values(*_halves(case, pages[:, :, i].transpose(1, 2))).reshape(b, hkv, n, d) for i in range(2))
    q = state["q"].float().mul(1 / math.sqrt(d)).view(b, t, hkv, group, d).transpose(1, 2).reshape(b, hkv, t * group, d)
    s = torch.matmul(q, k.transpose(2, 3).contiguous())
    del k
    if case["softcap"]:
        s = torch.tanh(s / case["softcap"]) * case["softcap"]
    seen = state["lens"].long()[:, None] - t + 1 + torch.arange(t, device="cuda")                # [b, t]
    hidden = torch.arange(n, device="cuda") >= seen.repeat_interleave(group, 1)[:, None, :, None]  # [b, 1, rows, n]
    s = s.masked_fill_(hidden, -math.inf)
    m = s.amax(-1, keepdim=True)
    s = s.sub_(m).exp_()
    total = s.sum(-1, keepdim=True)
    out = (torch.matmul(s, v) / total).view(b, hkv, t, group, d).transpose(1, 2).reshape(b, t, hq, d)
    lse = (m + torch.log(total)).view(b, hkv, t, group).transpose(2, 3).reshape(b, hq, t)
    return [out.to(state["q"].dtype), lse]


def _plain_fork(state):
    """Row i continues row parents[i]: its full pages are shared, its last one belongs
    to the first row that continues it and is copied for the others, and one more
    token has a page.  Free pages are taken from the lowest on, row by row."""
    case, page, pages = state["case"], state["case"]["page"], state["case"]["pages"]
    lens = state["lens"].long()[state["parents"].long()]
    table = state["table"].long()[state["parents"].long()]
    rows, entries = table.shape
    entry, row = torch.arange(entries, device="cuda")[None], torch.arange(rows, device="cuda")[:, None]
    full, partial = entry < lens[:, None] // page, (entry == lens[:, None] // page) & (lens[:, None] % page > 0)
    spare = lens.new_full((1,), pages)  # where the writes of the others go
    shared = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    shared[torch.where(full, table, spare).clamp_min(0)] = True
    last = torch.where(partial, table, spare)
    first = lens.new_full((pages + 1,), rows).scatter_reduce(0, last.reshape(-1), row.expand_as(last).reshape(-1), "amin")
    copied = partial & (shared[last] | (first[last] != row))
    fresh = copied | ((entry >= (lens[:, None] + page - 1) // page) & (entry < (lens[:, None] + page) // page))
    kept = full | (partial & ~copied)
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(kept, table, spare)] = True
    free = torch.argsort(used[:pages].int(), stable=True)  # the free pages first
    new = free[(fresh.reshape(-1).cumsum(0) - 1).clamp(0, pages - 1).view_as(table)]
    src, dst = table[copied], new[copied]
    for cache in state["caches"]:
        cache[dst] = cache[src]
    table = torch.where(kept, table, torch.where(fresh, new, -1))
    short = (fresh.sum() - (~used[:pages]).sum()).clamp_min(0).view(1)
    return [table.int(), lens.int(), short.int(), *state["caches"]]


def _plain_compact(state):
    pages, table = state["case"]["pages"], state["table"].long()
    used = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    used[torch.where(table >= 0, table, pages)] = True
    used = used[:pages]
    n, ids = used.sum(), torch.arange(pages, device="cuda")
    src, dst = ids[used & (ids >= n)], ids[~used & (ids < n)]
    place = ids.clone()
    place[src] = dst
    for cache in state["caches"]:
        cache[dst] = cache[src]
    table = torch.where(table >= 0, place[table.clamp_min(0)], -1)
    return [table.int(), n.view(1).int(), *state["caches"]]


def run(state):
    with torch.no_grad():
        if own:
            return list(_call(state))
        return {"store": _plain_store, "attention": _plain_attention, "fork": _plain_fork,
                "compact": _plain_compact}[state["case"]["op"]](state)


def work(case):
    if case["op"] in ("fork", "compact"):
        bytes_ = 2 * case["hkv"] * _page_bytes(case) * case["layers"]  # of a page
        if case["op"] == "compact":
            return {"bytes": 2 * _moved(case) * bytes_ + 8 * -(-case["used"] // case["entries"]) * case["entries"],
                    "flops": 0}
        copies = case["rows"] - case["rows"] // case["fanout"]
        return {"bytes": 2 * copies * bytes_ + 8 * case["rows"] * (case["entries"] + 3), "flops": 0}
    b, t, hkv, d, lens = case["batch"], case["tokens"], case["hkv"], case["hd"], _lens(case)
    key = 2 * hkv * (d // 2 + d // BLOCK)  # bytes of a key and its value
    if case["op"] == "store":
        tokens = sum(min(n, t) for n in lens)
        # read, stored, read again, and given back with the padding
        return {"bytes": tokens * (4 * hkv * d + 2 * key) + b * t * 4 * hkv * d + 4 * b, "flops": 0}
    pairs = sum(t * n - t * (t - 1) // 2 for n in lens)
    return {"bytes": 4 * b * t * case["hq"] * d + 4 * b * t * case["hq"] + key * sum(lens)
            + 4 * sum(-(-n // case["page"]) for n in lens) + 4 * b, "flops": 4 * case["hq"] * d * pairs}


# ---- the definitions in 64 bits, apart from the above -----------------------------

def _number(cache, case, page, kv, row):
    """Keys (kv 0) or values (1) [.., hkv, hd] of the rows `row` of pages `page`, in 64 bits."""
    half, blocks = case["hd"] // 2, case["hd"] // BLOCK
    where = row[..., None] * half + torch.arange(half, device="cuda")
    at = case["page"] * half + row[..., None] * blocks + torch.arange(blocks, device="cuda")
    head = torch.arange(case["hkv"], device="cuda")[:, None]
    codes = cache[page[..., None, None], kv, head, where[..., None, :]].long()
    scale = cache[page[..., None, None], kv, head, at[..., None, :]].double()
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    # E2M1: m / 2 for exponent 0, else (1 + m / 2) 2^(e - 1)
    e, m = (codes >> 1) & 3, (codes & 1).double() / 2
    v = torch.where(e == 0, m, (1 + m) * torch.exp2(e.double() - 1)) * (1 - 2 * (codes >> 3).double())
    return v * torch.exp2(scale - 127).repeat_interleave(BLOCK, -1)


def _exact_store(case, x):
    """Each value to the nearest of its block's numbers, ties to the even code."""
    grid = torch.tensor(VALUES, dtype=torch.float64, device="cuda")
    pos = x["lens"].long()[:, None] - case["tokens"] + torch.arange(case["tokens"], device="cuda")
    out = []
    for name in ("k", "v"):
        f = x[name].double().unflatten(-1, (-1, BLOCK))
        mantissa, exponent = torch.frexp(f.abs().amax(-1))        # mantissa in [0.5, 1)
        scale = torch.exp2((exponent - 3 + (mantissa >= 0.875).int()).clamp(LEAST - 127, MOST - 127).double())[..., None]
        y = f / scale
        low = (torch.searchsorted(grid, y.abs().contiguous(), right=True) - 1).clamp(0, 6)
        down, up = y.abs() - grid[low], grid[low + 1] - y.abs()
        near = torch.where((up < down) | ((up == down) & (low % 2 == 1)), low + 1, low)
        v = (grid[near] * y.sign() * scale).flatten(-2) * (pos >= 0)[..., None, None]
        out.append(v.clamp(-65504, 65504) if case["dtype"] == "f16" else v)
    return out


def _exact_attention(case, x):
    b, t, hq, hkv, d, page = (case[n] for n in ("batch", "tokens", "hq", "hkv", "hd", "page"))
    group, lens = hq // hkv, x["lens"].tolist()
    out = torch.empty(b, t, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.empty(b, hq, t, dtype=torch.float64, device="cuda")
    for i in range(b):
        key = torch.arange(lens[i], device="cuda")
        where = x["table"][i].long()[key // page]
        k, v = (_number(x["cache"], case, where, kv, key % page) for kv in range(2))  # [n, hkv, d]
        cut = torch.ones(t, lens[i], dtype=torch.bool, device="cuda").triu(lens[i] - t + 1)
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            for at in range(0, t, 128):  # tokens at a time
                q = x["q"][i, at:at + 128, heads].double()
                s = (q.reshape(-1, d) @ k[:, h].t().contiguous()).view(-1, group, lens[i]) / math.sqrt(d)
                if case["softcap"]:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                s = s.masked_fill(cut[at:at + 128, None], -math.inf)
                z = torch.logsumexp(s, -1)
                p = torch.exp(s - z[..., None])
                out[i, at:at + 128, heads] = (p.view(-1, lens[i]) @ v[:, h]).view(-1, group, d)
                lse[i, heads, at:at + 128] = z.t()
    return [out, lse]


def _exact_fork(case, x):
    page, pages = case["page"], case["pages"]
    old, parents = x["table"].tolist(), x["parents"].tolist()
    lens = [x["lens"].tolist()[p] for p in parents]
    table = [[-1] * len(old[0]) for _ in parents]
    full = {old[p][j] for p, n in zip(parents, lens) for j in range(n // page)}
    owner, wanted = {}, []
    for i, (p, n) in enumerate(zip(parents, lens)):
        table[i][: n // page] = old[p][: n // page]
        if n % page:
            last = old[p][n // page]
            if last in full or last in owner:
                wanted.append((i, n // page, last))
            else:
                owner[last] = i
                table[i][n // page] = last
        else:
            wanted.append((i, n // page, None))
    free = iter(sorted(set(range(pages)) - full - set(owner)))
    moves = []
    for i, j, source in wanted:
        table[i][j] = next(free)
        if source is not None:
            moves.append((source, table[i][j]))
    for source, target in moves:
        for cache in x["caches"]:
            cache[target].copy_(cache[source])
    return [torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
            torch.zeros(1, dtype=torch.int32).cuda(), *x["caches"]]


def _exact_compact(case, x):
    used = sorted({p for row in x["table"].tolist() for p in row if p >= 0})
    holes = sorted(set(range(len(used))) - set(used))
    place = {p: p for p in used}
    for source, target in zip([p for p in used if p >= len(used)], holes):
        place[source] = target
        for cache in x["caches"]:
            cache[target].copy_(cache[source])
    table = [[place.get(p, -1) for p in row] for row in x["table"].tolist()]
    return [torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor([len(used)], dtype=torch.int32).cuda(),
            *x["caches"]]


def exact(case, seed):
    """The operators' definitions, in 64 bits; pages and tables are whole numbers."""
    x = _inputs(case, seed)
    return {"store": _exact_store, "attention": _exact_attention, "fork": _exact_fork,
            "compact": _exact_compact}[case["op"]](case, x)
