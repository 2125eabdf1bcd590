"""A cache in pages of 4-bit numbers, its attention and its pages by their definitions, on
the CPU, numbers in 64 bits."""

import math

import pytest
import torch

CODES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def numbers(cache, dim):
    """float64 [pages, 2, hkv, page_size, dim]."""
    row = dim // 2 + dim // 32
    size = cache.shape[-1] // row
    codes = cache[..., : size * dim // 2].unflatten(-1, (size, dim // 2)).long()
    scale = cache[..., size * dim // 2:].unflatten(-1, (size, dim // 32)).double()
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = CODES[codes & 7] * (1 - 2 * (codes >> 3).double())
    scale = torch.where(scale > 252, math.nan, torch.exp2(scale - 127))
    return v * scale.repeat_interleave(32, -1)


def nearest(x):
    """What a cache holds of [.., dim] values: each block's power of two, each value its
    nearest number, by trying all of them."""
    f = x.double().unflatten(-1, (-1, 32))
    top = f.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -100)
    for i in range(-100, 126):  # the smallest power whose sevenfold is past the largest value
        e = torch.where((top >= 7 * 2.0 ** (i - 1)), torch.full_like(e, i), e)
    scale = torch.exp2(e)
    far = (f.abs() / scale).unsqueeze(-1)
    gap = (far.clamp_max(6) - CODES).abs()
    # ties to the even code: an odd one loses by a hair
    code = (gap + torch.tensor([0, 1e-9] * 4, dtype=torch.float64)).argmin(-1)
    v = CODES[code] * f.sign() * scale
    return torch.where(top.isfinite(), v, math.nan).flatten(-2)


def same(a, b):
    """Equal numbers, and NaN in the same places."""
    a, b = a.cpu().double(), b.cpu().double()
    assert a.shape == b.shape
    bad = ~((a == b) | (a.isnan() & b.isnan()))
    if bool(bad.any()):
        at = tuple(bad.nonzero()[0].tolist())
        pytest.fail(f"{int(bad.sum())} of {bad.numel()} differ, first at {at}: {a[at]} for {b[at]}")


def sequence(v, table, length):
    """Keys and values [keys, hkv, dim] of a row of the table, and which of them there are, from the
    cache's numbers."""
    size = v.shape[3]
    n = min(max(int(length), 0), len(table) * size)
    pages = [int(table[x // size]) for x in range(n)]
    there = torch.tensor([0 <= p < v.shape[0] for p in pages], dtype=torch.bool)
    where = torch.tensor([p if 0 <= p < v.shape[0] else 0 for p in pages], dtype=torch.long)
    rows = torch.arange(n) % size
    return v[where, 0, :, rows], v[where, 1, :, rows], there


def attention(q, cache, table, lens, scale, cap=0.0):
    """out [B, T, Hq, D] and lse [B, Hq, T], with their tolerances.

    Keys and values are exact in the products, as are queries.  A score is a sum of D products in
    FP32 (2 D for FP16 queries, which are two terms): off by at most 2 D 2^-24 sum |q k| scale, with a
    softcap 4e-7 cap more (its tanh is within 2^-21 of 1); 1e-5 covers the exponent's rounding and
    its instruction: d in all.  A probability in two BF16 terms is off by r = 2^-8 2^-8 of itself; BF16
    queries with more than 32 rows to a KV head (T Hq / Hkv) have one term, r = 2^-8, half a step.  The
    sums over n keys are off by n 2^-23, twice that with the join of parts.  So an output is off by
    (r + 2 d + n 2^-22) sum p |v| and half a step of its type, lse by d + n 2^-22 + 1e-6 |lse|."""
    b, t, hq, d = q.shape
    u = torch.finfo(q.dtype).eps / 2
    least = torch.finfo(q.dtype).smallest_normal * u  # half a step of what is not normal
    out, tol_o = (torch.zeros(b, t, hq, d, dtype=torch.float64) for _ in range(2))
    lse, tol_l = torch.full((b, hq, t), -math.inf, dtype=torch.float64), torch.zeros(b, hq, t, dtype=torch.float64)
    group = hq // cache.shape[2]
    r = 2.0 ** -8 if q.dtype == torch.bfloat16 and t * group > 32 else 2.0 ** -16
    held = numbers(cache, d)
    for i in range(b):
        k, v, there = sequence(held, table[i].tolist(), lens[i])
        for j in range(t):
            c = max(0, min(max(int(lens[i]), 0) - t + j + 1, k.shape[0]))
            if not there[:c].any():
                continue
            kk, vv = (x[:c][there[:c]].repeat_interleave(group, 1) for x in (k, v))  # [n, hq, d]
            x = q[i, j].double()
            s = (kk * x).sum(-1) * scale
            err = (kk * x).abs().sum(-1).nan_to_num(0).amax(0) * scale * 2 * d * 2.0 ** -24 + 1e-5
            if cap:
                s = cap * torch.tanh(s / cap)
                err = err + 4e-7 * cap
            z = torch.logsumexp(s, 0)
            p = torch.exp(s - z)
            out[i, j] = (p[..., None] * vv).sum(0)
            lse[i, :, j] = z
            size = (p[..., None] * vv.abs()).sum(0)
            tol_o[i, j] = (r + 2 * err + c * 2.0 ** -22)[:, None] * size + out[i, j].abs() * u * 1.01 + least
            tol_l[i, :, j] = err + c * 2.0 ** -22 + 1e-6 * z.abs()
    return out, lse, tol_o, tol_l


def attention_at_scale(q, cache, table, lens, scale, cap=0.0):
    """The same of whole sequences whose pages are all there, on the operands' device."""
    b, t, hq, d = q.shape
    u, group = torch.finfo(q.dtype).eps / 2, hq // cache.shape[2]
    least = torch.finfo(q.dtype).smallest_normal * u  # half a step of what is not normal
    r = 2.0 ** -8 if q.dtype == torch.bfloat16 and t * group > 32 else 2.0 ** -16
    out, tol_o = (torch.zeros(b, t, hq, d, dtype=torch.float64, device=q.device) for _ in range(2))
    lse, tol_l = (torch.zeros(b, hq, t, dtype=torch.float64, device=q.device) for _ in range(2))
    half, size = d // 2, cache.shape[-1] // (d // 2 + d // 32)
    lut = torch.cat([CODES, -CODES]).to(q.device)
    for i in range(b):
        n = int(lens[i])
        pages = table[i, : -(-n // size)].long()
        hidden = torch.arange(n, device=q.device) > n - t + torch.arange(t, device=q.device)[:, None]  # [t, n]
        for h in range(cache.shape[2]):
            kv = []
            for x in cache[pages, :, h].unbind(1):
                codes = x[:, : size * half].reshape(-1, half)[:n].long()
                scale2 = torch.exp2(x[:, size * half:].reshape(-1, d // 32)[:n].double() - 127)
                kv.append(lut[torch.stack([codes & 15, codes >> 4], -1).flatten(1)] * scale2.repeat_interleave(32, 1))
            k, v = kv
            heads = slice(h * group, (h + 1) * group)
            x = q[i, :, heads].reshape(-1, d).double()
            s = (x @ k.t().contiguous() * scale).view(t, group, n)
            err = (x.abs() @ k.abs().t().contiguous()).amax(1).view(t, group) * scale * 2 * d * 2.0 ** -24 + 1e-5
            if cap:
                s, err = cap * torch.tanh(s / cap), err + 4e-7 * cap
            s = s.masked_fill(hidden[:, None], -math.inf)
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - z[..., None])
            out[i, :, heads] = (p.view(-1, n) @ v).view(t, group, d)
            total = (p.view(-1, n) @ v.abs()).view(t, group, d)
            lse[i, heads] = z.t()
            tol_o[i, :, heads] = (r + 2 * err + n * 2.0 ** -22)[..., None] * total + out[i, :, heads].abs() * u * 1.01 + least
            tol_l[i, heads] = (err + n * 2.0 ** -22 + 1e-6 * z.abs()).t()
    return tuple(x.cpu() for x in (out, lse, tol_o, tol_l))


def check(got, want):
    """An attention's results within their tolerances; rows and elements that are no numbers alike."""
    out, lse, tol_o, tol_l = want
    o, z = got[0].cpu().double(), got[1].cpu().double()
    assert got[1].dtype == torch.float32 and o.shape == out.shape and z.shape == lse.shape
    assert torch.equal(o.isnan(), out.isnan()) and torch.equal(z.isnan(), lse.isnan())
    assert torch.equal(z == -math.inf, lse == -math.inf)
    off = ((o - out).abs() - tol_o).nan_to_num(-1)
    assert bool((off <= 0).all()), float(off.max())
    off = ((z - lse).abs() - tol_l).nan_to_num(-1)  # Inf - Inf too
    assert bool((off <= 0).all()), float(off.max())


def fork(table, lens, parents, tokens, size, pages):
    """New table, lengths, pages wanted and not there, and (source, target) of each copy."""
    entries = table.shape[1]
    old = [[p if 0 <= p < pages else -1 for p in row] for row in table.tolist()]
    parents = list(range(len(old))) if parents is None else parents.tolist()
    rows, full, owner = [], set(), {}
    for i, p in enumerate(parents):
        ok = 0 <= p < len(old)
        n = min(max(int(lens[p]), 0), entries * size) if ok else 0
        rows.append((old[p] if ok else [-1] * entries, n, ok))
        full |= {x for x in rows[-1][0][: n // size] if x >= 0}
    for i, (row, n, _) in enumerate(rows):
        if n % size and row[n // size] >= 0:
            owner.setdefault(row[n // size], i)
    free = iter(sorted(set(range(pages)) - full - set(owner)))
    out, moves, short = torch.full((len(rows), entries), -1, dtype=torch.int32), [], 0
    for i, (row, n, ok) in enumerate(rows):
        for j in range(n // size):
            out[i, j] = row[j]
        wanted = []
        if n % size:
            last = row[n // size]
            if last < 0:
                short += tokens > 0
            elif last in full or owner[last] != i:
                wanted.append((n // size, last))
            else:
                out[i, n // size] = last
        if ok:
            wanted += [(j, None) for j in range(-(-n // size), -(-(n + tokens) // size))]
        for j, source in wanted:
            page = next(free, None) if j < entries else None
            if page is None:
                short += 1
                continue
            out[i, j] = page
            if source is not None:
                moves.append((source, page))
    return out, torch.tensor([n for _, n, _ in rows], dtype=torch.int32), short, moves


def compact(table, pages):
    """New table, pages in use, and (source, target) of each copy."""
    used = sorted({p for p in table.flatten().tolist() if 0 <= p < pages})
    holes = sorted(set(range(len(used))) - set(used))
    moves = list(zip([p for p in used if p >= len(used)], holes))
    place = {p: p for p in used} | dict(moves)
    out = [[place.get(p, -1) for p in row] for row in table.tolist()]
    return torch.tensor(out, dtype=torch.int32).view(table.shape), len(used), moves
