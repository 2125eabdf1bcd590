"""Attention over a cache in pages of 4-bit numbers against its definition in 64 bits
(paged_reference.attention derives the tolerances)."""

import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

# dtype, batch, tokens, hq, hkv, dim, page_size, cap, lens
CASES = [
    ("bf16", 1, 1, 1, 1, 128, 16, 0.0, [1]),
    ("bf16", 2, 1, 4, 1, 128, 64, 0.0, [5, 64]),
    ("f16", 3, 1, 8, 2, 64, 32, 0.0, [70, 0, 33]),
    ("f16", 2, 1, 4, 4, 128, 16, 30.0, [64, 65]),
    ("bf16", 5, 1, 8, 1, 64, 128, 50.0, [300, 1, 2, 299, 128]),
    ("bf16", 9, 1, 16, 4, 128, 16, 0.0, [40, 0, 1, 39, 7, 32, 33, 31, 16]),
    ("f16", 2, 7, 10, 2, 64, 48, 0.0, [50, 3]),           # 35 rows; tokens that see nothing
    ("bf16", 3, 33, 4, 4, 128, 16, 0.0, [90, 33, 34]),
    ("bf16", 1, 150, 2, 1, 128, 64, 30.0, [150]),
    ("f16", 2, 40, 8, 2, 128, 32, 0.0, [64, 40]),
    ("bf16", 2, 3, 4, 2, 64, 16, 0.0, [10, 1]),
    ("bf16", 3, 2, 6, 3, 64, 16, 0.0, [-5, 1000, 30]),    # a length past the table
    ("bf16", 2, 1, 32, 8, 128, 64, 0.0, [3000, 2950]),    # sequences that several blocks share
    ("bf16", 1, 1, 8, 1, 128, 16, 0.0, [9000]),
    ("f16", 1, 4, 64, 8, 64, 32, 20.0, [5000]),
    ("bf16", 2, 1, 64, 1, 128, 64, 0.0, [700, 129]),      # 64 heads to a KV head
]


def make(case, seed=0, entries=None):
    """q, cache, table and lens on the CPU; pages in any order, what lies past a sequence NaN."""
    dtype, b, t, hq, hkv, dim, size, cap, lens = case
    g = torch.Generator().manual_seed(seed)
    counts = [-(-max(0, min(n, 64 * size if n == 1000 else n)) // size) for n in lens]
    counts = [min(n, 3) if lens[i] == 1000 else n for i, n in enumerate(counts)]
    entries = entries or max(1, max(counts))
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g)
    table, at = torch.full((b, entries), -1, dtype=torch.int32), 0
    cache = torch.randint(0, 256, (pages, 2, hkv, size * (dim // 2 + dim // 32)), generator=g, dtype=torch.uint8)
    codes = size * dim // 2
    cache[..., codes:] = cache[..., codes:] % 5 + 123
    for i, n in enumerate(counts):
        table[i, :n] = order[at: at + n]
        at += n
        if n and 0 < lens[i] < n * size:
            first = codes + (lens[i] - (n - 1) * size) * (dim // 32)
            cache[order[at - 1], :, :, first:] = 255
    q = (torch.randn(b, t, hq, dim, generator=g) * (8 if cap else 2)).to(torch.bfloat16 if dtype == "bf16" else torch.float16)
    return q, cache, table, torch.tensor(lens, dtype=torch.int32)


def run(t, cuda, **args):
    from sfu_repro import fa4_runtime

    return fa4_runtime.flash_attn_paged_fp4(*(x.to(cuda) for x in t), **args)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:8])))
def test_attention(cuda, case):
    t = make(case)
    ref.check(run(t, cuda, softcap=case[7]), ref.attention(*t, 1 / math.sqrt(case[5]), case[7]))


def test_scale(cuda):
    t = make(CASES[6], seed=2)
    ref.check(run(t, cuda, softmax_scale=0.03), ref.attention(*t, 0.03))


def test_scores_of_any_size(cuda):
    """Scores of several thousand that rise and fall along the keys, so that the maximum
    moves in every part; all equal; and beyond 2^20."""
    q, cache, table, lens = make(("bf16", 3, 1, 4, 2, 128, 32, 0.0, [2000, 513, 0]), seed=3)
    t = (q * 500, cache, table, lens)
    ref.check(run(t, cuda), ref.attention(*t, 1 / math.sqrt(128)))
    t = (q * 0, cache, table, lens)
    ref.check(run(t, cuda), ref.attention(*t, 1 / math.sqrt(128)))
    t = (q * 2.0 ** 24, cache, table, lens)
    ref.check(run(t, cuda), ref.attention(*t, 1 / math.sqrt(128)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_every_exponent(cuda, dtype, dim):
    """Blocks from 2^-100 to 2^125 beside each other: in values, and in keys whose scores stay finite."""
    q, cache, table, lens = make((dtype, 2, 1, 4, 2, dim, 16, 0.0, [300, 77]), seed=4)
    codes = 16 * dim // 2
    g = torch.Generator().manual_seed(5)
    for page in range(cache.shape[0]):
        n = cache[page, 1, :, codes:].numel()
        cache[page, 1, :, codes:] = torch.randint(27, 253, (n,), generator=g, dtype=torch.uint8).view(2, -1)
        cache[page, 0, :, codes:] = torch.randint(27, 131, (n,), generator=g, dtype=torch.uint8).view(2, -1)
    t = (q, cache, table, lens)
    out, lse, tol_o, tol_l = ref.attention(*t, 1 / math.sqrt(dim))
    got = run(t, cuda)
    most = float(torch.finfo(q.dtype).max)
    # what passes the result's type, or comes close to it, in any finite or infinite form
    far = out.abs() + tol_o >= most * 0.99
    assert bool((got[0].cpu().double().abs() >= most * 0.97)[far].all())
    o, z = got[0].cpu().double(), got[1].cpu().double()
    assert bool(((o - out).abs() <= tol_o)[~far].all()) and bool(((z - lse).abs() <= tol_l).all())


def test_fp16_queries_of_any_size(cuda):
    """An FP16 query is two BF16 terms, exactly: largest and smallest numbers, those that BF16 lacks."""
    q, cache, table, lens = make(("f16", 2, 2, 8, 2, 128, 16, 0.0, [200, 77]), seed=6)
    q[0, 0] = torch.randint(0, 0x7c00, q[0, 0].shape, generator=torch.Generator().manual_seed(7)).to(torch.int16).view(torch.float16)
    q[0, 1] = 65504.0 * torch.randn(q[0, 1].shape, generator=torch.Generator().manual_seed(8)).sign()
    q[1, 0] = 2.0 ** -24
    q[1, 1] = 1 + 2.0 ** -10
    for scale in (2.0 ** -20, 2.0 ** -4):
        t = (q, cache, table, lens)
        ref.check(run(t, cuda, softmax_scale=scale), ref.attention(*t, scale))


# dtype, tokens, hq, hkv, dim: one tile of 16 rows, of 32, several
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("case", [("bf16", 3, 4, 2, 128), ("f16", 5, 4, 1, 64), ("bf16", 25, 4, 2, 64),
                                  ("f16", 40, 2, 1, 128)], ids=lambda c: "-".join(map(str, c)))
def test_what_other_tokens_see(cuda, case, cap):
    """Blocks that are no numbers, ahead of the token that brings them: that token and those
    behind it get NaN, in a value's elements or in the whole row for a key; the others the same bits."""
    from sfu_repro import fa4_runtime

    dtype, tokens, hq, hkv, dim = case
    t = [x.to(cuda) for x in make((dtype, 2, tokens, hq, hkv, dim, 16, cap, [90, 88]))]
    q, cache, table, lens = t
    clean = fa4_runtime.flash_attn_paged_fp4(*t, softcap=cap)
    assert bool(clean[0].isfinite().all())
    h, codes = hkv - 1, 16 * dim // 2
    heads = slice(h * hq // hkv, None)
    keep = cache.clone()
    for what, bytes_ in ((1, (253, 255)), (0, (254, 255))):
        cache.copy_(keep)
        for b in range(2):
            for late, byte in ((2, bytes_[0]), (1, bytes_[1])):  # the token before the last, and the last
                x = int(lens[b]) - late
                cache[int(table[b, x // 16]), what, h, codes + x % 16 * (dim // 32) + late - 1] = byte
        bad = fa4_runtime.flash_attn_paged_fp4(*t, softcap=cap)
        want, lse = clean[0].clone(), clean[1].clone()
        if what == 1:
            want[:, tokens - 2:, heads, 32:64] = math.nan
            want[:, tokens - 1:, heads, :32] = math.nan
        else:
            want[:, tokens - 2:, heads], lse[:, heads, tokens - 2:] = math.nan, math.nan
        ref.same(bad[0], want)
        ref.same(bad[1], lse)


def test_values_that_all_see(cuda):
    """A block that is no number far ahead of every token: NaN for all of its head's rows."""
    t = make(("bf16", 2, 3, 4, 2, 128, 16, 0.0, [300, 200]), seed=9)
    q, cache, table, lens = t
    codes = 16 * 64
    cache[int(table[0, 1]), 1, 1, codes + 5 * 4 + 2] = 255
    want = ref.attention(*t, 1 / math.sqrt(128))
    assert bool(want[0][0, :, 2:, 64:96].isnan().all()) and int(want[0].isnan().sum()) == 3 * 2 * 32
    ref.check(run(t, cuda), want)


def test_queries_that_are_no_numbers(cuda):
    """They reach their own rows alone; an infinite one takes what its scores make of it."""
    for dtype in ("bf16", "f16"):
        t = list(make((dtype, 2, 3, 8, 2, 64, 16, 0.0, [100, 64]), seed=10))
        clean = run(t, cuda)
        t[0] = t[0].clone()
        t[0][0, 1, 3, 7], t[0][1, 2, 0, 0] = math.nan, math.inf
        got = run(t, cuda)
        assert bool(got[0][0, 1, 3].isnan().all()) and bool(got[1][0, 3, 1].isnan())
        same = torch.ones(2, 3, 8, dtype=torch.bool)
        same[0, 1, 3] = same[1, 2, 0] = False
        assert torch.equal(got[0][same], clean[0][same])
        assert torch.equal(got[1].transpose(1, 2)[same], clean[1].transpose(1, 2)[same])
        assert not bool(got[0][1, 2, 0].isfinite().any())


def test_pages_that_are_not_there(cuda):
    """Entries that name no page, inside a sequence, at its start and all along it; numbers outside the cache."""
    for dtype, tokens, dim in (("bf16", 1, 128), ("f16", 4, 64), ("bf16", 30, 128)):
        t = make((dtype, 3, tokens, 4, 2, dim, 16, 0.0, [300, 90, 70]), seed=11)
        table = t[2]
        table[0, 0], table[0, 5], table[0, 6], table[1, 5] = -1, 2 ** 31 - 1, t[1].shape[0], -2 ** 31
        table[2] = -1
        ref.check(run(t, cuda), ref.attention(*t, 1 / math.sqrt(dim)))


def test_lengths_of_any_value(cuda):
    """Past the table, negative, the ends of int32: the keys that there are."""
    t = list(make(("bf16", 4, 2, 4, 2, 128, 16, 0.0, [64, 64, 64, 64]), seed=12))
    t[3] = torch.tensor([2 ** 31 - 1, -2 ** 31, 65, 66], dtype=torch.int32)
    ref.check(run(t, cuda), ref.attention(*t, 1 / math.sqrt(128)))


def test_layouts(cuda):
    """A query view of a packed projection, one that has to be copied, tables and lengths that
    are views: the same bits."""
    from sfu_repro import fa4_runtime

    t = [x.to(cuda) for x in make(("bf16", 3, 2, 8, 2, 128, 32, 0.0, [40, 2, 170]))]
    want = fa4_runtime.flash_attn_paged_fp4(*t)
    q, cache, table, lens = t
    packed = torch.zeros(3, 2, 24, 128, dtype=q.dtype, device=cuda)
    packed[:, :, 4:12] = q
    odd = torch.zeros(3, 2, 8, 129, dtype=q.dtype, device=cuda)
    odd[..., 1:] = q
    wide = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device=cuda)
    wide[:, : table.shape[1]] = table
    for other in ((packed[:, :, 4:12], cache, wide[:, : table.shape[1]], torch.stack([lens, lens], 1)[:, 0]),
                  (odd[..., 1:], cache, table.t().contiguous().t(), lens), (q, cache, wide, lens)):
        got = fa4_runtime.flash_attn_paged_fp4(*other)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = fa4_runtime.flash_attn_paged_fp4(q[:1].expand(3, -1, -1, -1), cache, table[:1].expand(3, -1), lens[:1].expand(3))
    alone = fa4_runtime.flash_attn_paged_fp4(q[:1], cache, table[:1], lens[:1])
    assert all(float((o - a).float().abs().max()) < 0.02 for o, a in zip(one, alone))


def test_order_of_pages_and_page_size_make_no_difference(cuda):
    """The same keys in pages of 16 and 64, in other places: the same bits."""
    from sfu_repro import fa4_runtime

    q, cache, table, lens = (x.to(cuda) for x in make(("bf16", 2, 1, 8, 2, 128, 64, 0.0, [500, 130]), seed=13))
    want = fa4_runtime.flash_attn_paged_fp4(q, cache, table, lens)
    n, codes = cache.shape[0], 64 * 64
    parts = [cache[..., :codes].unflatten(-1, (4, 16 * 64)), cache[..., codes:].unflatten(-1, (4, 16 * 4))]
    small = torch.cat(parts, -1).permute(0, 3, 1, 2, 4).reshape(4 * n, 2, 2, -1)
    order = torch.randperm(4 * n, generator=torch.Generator().manual_seed(1)).to(cuda)
    moved = torch.empty_like(small)
    moved[order] = small
    entries = torch.where(table[..., None] >= 0, table[..., None] * 4 + torch.arange(4, device=cuda), 0).flatten(1)
    entries = order[entries.long()].to(torch.int32)
    got = fa4_runtime.flash_attn_paged_fp4(q, moved, entries, lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits(cuda):
    """Pages behind the first 2^32 bytes of a cache."""
    from sfu_repro import fa4_runtime

    t = make(("bf16", 2, 1, 4, 2, 128, 64, 0.0, [500, 100]), seed=14)
    want = run(t, cuda)
    pages, first = t[1].shape[0], 2 ** 33 // t[1][0].numel()
    far = torch.empty(first + pages, *t[1].shape[1:], dtype=torch.uint8, device=cuda)
    far[first:] = t[1].to(cuda)
    got = fa4_runtime.flash_attn_paged_fp4(t[0].to(cuda), far, (t[2] + first * (t[2] >= 0)).to(torch.int32).to(cuda), t[3].to(cuda))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dim", [64, 128])
def test_d4_softcap_is_the_prefix_attentions(cuda, dim):
    """The D4 program over what the cache holds, as the shared-prefix attention computes it from
    the same numbers in BF16: its scores are the same up to the order of a product's sum, which may
    move a BF16 score by a step (2^-8 of 50), so results by a quarter, and their mean by far less."""
    from sfu_repro import fa4_runtime, paged_cache

    q, cache, table, lens = (x.to(cuda) for x in make(("bf16", 3, 2, 8, 2, dim, 16, 0.0, [300, 17, 64]), seed=15))
    q = q * 4
    mod = fa4_runtime.create_softcap_scoremod_backend(50.0, 4)
    out, lse = fa4_runtime.flash_attn_paged_fp4(q, cache, table, lens, score_mod=mod)
    n = int(lens.max())
    for b in range(3):
        k, v = paged_cache.load_fp4(cache, table[b:b + 1], lens[b:b + 1], int(lens[b]), dim)
        want, want_lse = fa4_runtime.flash_attn_shared_prefix(q[b:b + 1], k[0, :0], v[0, :0], k, v, lens[b:b + 1],
                                                              score_mod=mod)
        size = float(v.float().abs().max())
        assert float((out[b:b + 1].float() - want.float()).abs().max()) <= 0.25 * size
        assert float((out[b:b + 1].float() - want.float()).abs().mean()) <= 2.0 ** -8 * size
        assert float((lse[b:b + 1] - want_lse).abs().max()) <= 0.25
    assert n == 300


def test_equals_shared_prefix_attention_without_prefix(cuda):
    """Both compute the same softmax of the same numbers; the other rounds P in two terms too."""
    from sfu_repro import fa4_runtime, paged_cache

    q, cache, table, lens = (x.to(cuda) for x in make(("bf16", 2, 2, 8, 2, 128, 32, 0.0, [500, 77]), seed=16))
    out, lse = fa4_runtime.flash_attn_paged_fp4(q, cache, table, lens)
    for b in range(2):
        k, v = paged_cache.load_fp4(cache, table[b:b + 1], lens[b:b + 1], int(lens[b]), 128)
        want, want_lse = fa4_runtime.flash_attn_shared_prefix(q[b:b + 1], k[0, :0], v[0, :0], k, v, lens[b:b + 1])
        assert float((out[b:b + 1].float() - want.float()).abs().max()) <= 2 * 2.0 ** -8 * float(v.float().abs().max())
        assert float((lse[b:b + 1] - want_lse).abs().max()) <= 1e-4


def test_many_sequences(cuda):
    """More sequences than a block has threads, among them empty ones; more rows of tiles than blocks."""
    lens = [(i * 37) % 130 for i in range(700)]
    t = make(("bf16", 700, 1, 4, 2, 64, 16, 0.0, lens), seed=17)
    ref.check(run(t, cuda), ref.attention(*t, 1 / 8))
    t = make(("bf16", 20, 70, 2, 2, 64, 16, 0.0, [70 + i for i in range(20)]), seed=18)
    ref.check(run(t, cuda), ref.attention(*t, 1 / 8))


def test_empty_calls(cuda):
    from sfu_repro import fa4_runtime

    q, cache, table, lens = (x.to(cuda) for x in make(CASES[1]))
    out, lse = fa4_runtime.flash_attn_paged_fp4(q[:0], cache, table[:0], lens[:0])
    assert out.shape == (0, 1, 4, 128) and lse.shape == (0, 4, 1)
    out, lse = fa4_runtime.flash_attn_paged_fp4(q[:, :0], cache, table, lens)
    assert out.shape == (2, 0, 4, 128) and lse.shape == (2, 4, 0)
    for c, tab in ((cache[:0], table), (cache, table[:, :0])):
        out, lse = fa4_runtime.flash_attn_paged_fp4(q, c, tab, lens)
        assert not bool(out.any()) and bool((lse == -math.inf).all())


def test_repeats_and_streams(cuda):
    """The same bits on every call, on another stream, and from two streams at once."""
    from sfu_repro import fa4_runtime

    t = [x.to(cuda) for x in make(("bf16", 3, 2, 32, 8, 128, 64, 0.0, [2000, 700, 1]), seed=19)]
    u = [x.to(cuda) for x in make(("f16", 2, 1, 16, 4, 64, 16, 0.0, [1500, 1]), seed=20)]
    want, other = fa4_runtime.flash_attn_paged_fp4(*t), fa4_runtime.flash_attn_paged_fp4(*u)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(8):
        for i, (s, x) in enumerate(zip(streams, (t, u))):
            with torch.cuda.stream(s):
                got[i].append(fa4_runtime.flash_attn_paged_fp4(*x))
    torch.cuda.synchronize()
    for results, w in zip(got, (want, other)):
        assert all(torch.equal(a, b) for r in results for a, b in zip(r, w))


def test_graph(cuda):
    """Captured calls follow the table, the lengths and the cache from replay to replay."""
    from sfu_repro import fa4_runtime

    cases = [make(("bf16", 3, 2, 8, 2, 128, 32, 0.0, lens), seed=s, entries=40) for s, lens in
             enumerate(([1200, 2, 33], [5, 0, 1000], [1, 1, 1], [1200, 2, 33]))]
    pages = max(c[1].shape[0] for c in cases)
    static = [cases[0][0].to(cuda), torch.zeros(pages, *cases[0][1].shape[1:], dtype=torch.uint8, device=cuda),
              cases[0][2].to(cuda), cases[0][3].to(cuda)]
    fa4_runtime.flash_attn_paged_fp4(*static)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = fa4_runtime.flash_attn_paged_fp4(*static)
    for case in cases:
        for s, x in zip(static, case):
            s[: x.shape[0]] = x.to(cuda)
        g.replay()
        want = fa4_runtime.flash_attn_paged_fp4(*static)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        ref.check((out, lse), ref.attention(case[0], static[1].cpu(), case[2], case[3], 1 / math.sqrt(128)))


def test_refusals(cuda):
    from sfu_repro import fa4_runtime

    q, cache, table, lens = (x.to(cuda) for x in make(CASES[1]))
    call = fa4_runtime.flash_attn_paged_fp4
    with pytest.raises(RuntimeError, match="no backward"):
        call(q.clone().requires_grad_(True), cache, table, lens)
    for bad, message in (((q.float(), cache, table, lens), "float16 or bfloat16"),
                         ((q[0], cache, table, lens), "must have shape"),
                         ((q[..., :96], cache, table, lens), "head_dim must be 64 or 128"),
                         ((q[..., :64], cache[..., :-16], table, lens), "contiguous"),
                         ((q[..., :64], cache, table, lens), None),
                         ((q, cache[..., :-64].contiguous(), table, lens), "whole multiples"),
                         ((q, cache.view(torch.int8), table, lens), "uint8"),
                         ((q, cache.cpu(), table, lens), "CUDA"),
                         ((q, cache, table.long(), lens), "table must be int32"),
                         ((q, cache, table, lens.long()), "lens must be int32"),
                         ((q, cache, table.cpu(), lens), "same CUDA device"),
                         ((q, cache, table[:1], lens[:1]), "batch"),
                         ((q, cache, table, lens[:1]), "lens must have shape"),
                         ((q[:, :, :0], cache, table, lens), "positive multiple")):
        if message is None:  # pages of 64 rows of 128 elements are pages of 128 rows of 64
            call(*bad)
            continue
        with pytest.raises(RuntimeError, match=message):
            call(*bad)
    with pytest.raises(RuntimeError, match="softmax_scale"):
        call(q, cache, table, lens, softmax_scale=0.0)
    with pytest.raises(NotImplementedError):
        call(q, cache, table, lens, exp2_emu_freq=16)
    with pytest.raises(TypeError, match="bfloat16 program"):
        call(q.half(), cache, table, lens, score_mod=fa4_runtime.create_softcap_scoremod_backend(30.0))
