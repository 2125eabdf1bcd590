"""The cache in pages of 4-bit numbers at the sizes of large calls, against the definition in 64 bits."""

import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

# dtype, tokens, hq, hkv, dim, page_size, cap, lens
CASES = [
    ("bf16", 1, 8, 1, 64, 64, 0.0, [131071]),             # one unit in many pieces
    ("f16", 1, 8, 2, 128, 16, 50.0, [40000, 129]),
    ("bf16", 1, 4, 1, 128, 128, 0.0, [600000]),
    ("bf16", 1, 32, 8, 128, 64, 0.0, [16384 * i // 15 + 1 for i in range(16)]),
    ("bf16", 1, 32, 32, 64, 32, 30.0, [1000 + 37 * i for i in range(40)]),
    ("bf16", 5, 32, 4, 128, 64, 0.0, [4100, 5, 2000, 4099, 77, 1024]),
    ("f16", 3, 32, 8, 64, 48, 0.0, [9000, 500]),
    ("bf16", 512, 32, 8, 128, 64, 0.0, [2500, 512]),
    ("f16", 300, 8, 2, 128, 64, 30.0, [3000, 301]),
    ("bf16", 1000, 4, 4, 64, 16, 0.0, [1000, 2047, 1001]),
    ("bf16", 1, 16, 1, 128, 64, 0.0, [3000] * 40),
    ("bf16", 16, 8, 4, 64, 64, 20.0, [8191] * 3),         # 32 rows
]


def _make(case, device, seed=0):
    dtype, t, hq, hkv, dim, size, cap, lens = case
    g = torch.Generator(device=device).manual_seed(seed)
    counts = [-(-n // size) for n in lens]
    order = torch.randperm(sum(counts) + 2, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table, at = torch.full((len(lens), max(counts) + 1), -1, dtype=torch.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at: at + n]
        at += n
    cache = torch.randint(0, 256, (order.numel(), 2, hkv, size * (dim // 2 + dim // 32)), generator=g, device=device,
                          dtype=torch.uint8)
    codes = size * dim // 2
    cache[..., codes:] = cache[..., codes:] % 4 + 123
    q = torch.randn(len(lens), t, hq, dim, generator=g, device=device) * (8 if cap else 1.5)
    return (q.to(torch.bfloat16 if dtype == "bf16" else torch.float16), cache, table.to(device),
            torch.tensor(lens, dtype=torch.int32, device=device))


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
def test_attention(cuda, case):
    from sfu_repro import fa4_runtime

    t = _make(case, cuda)
    got = fa4_runtime.flash_attn_paged_fp4(*t, softcap=case[6])
    ref.check(got, ref.attention_at_scale(*t, 1 / math.sqrt(case[4]), case[6]))
    again = fa4_runtime.flash_attn_paged_fp4(*t, softcap=case[6])
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_a_wide_table_costs_nothing_but_its_rows(cuda):
    """Entries behind the keys, and how many there are, change no bit of the result."""
    from sfu_repro import fa4_runtime

    q, cache, table, lens = _make(("bf16", 1, 32, 8, 128, 64, 0.0, [3000, 17, 900]), cuda)
    want = fa4_runtime.flash_attn_paged_fp4(q, cache, table, lens)
    wide = torch.full((3, 2 ** 14), 2 ** 31 - 1, dtype=torch.int32, device=cuda)
    wide[:, : table.shape[1]] = table
    got = fa4_runtime.flash_attn_paged_fp4(q, cache, wide, lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_store_and_load_of_a_long_prompt(cuda, dtype):
    """Every element of 2 x 8000 tokens is within half a step of its block's numbers: the step
    between 4 and 6 is 2, so at most a power of two that is at most 2 / 7 of the block's largest."""
    from sfu_repro import paged_cache

    g = torch.Generator(device=cuda).manual_seed(3)
    k, v = (torch.randn(2, 8000, 6, 128, generator=g, device=cuda, dtype=dtype) * 3 for _ in range(2))
    cache = paged_cache.fp4_cache(260, 6, 128, 64, device=cuda)
    table = torch.randperm(260, generator=torch.Generator().manual_seed(1))[:250].view(2, 125).to(torch.int32).to(cuda)
    lens = torch.full((2,), 8000, dtype=torch.int32, device=cuda)
    paged_cache.store_fp4(cache, k, v, table, lens)
    for x, y in zip((k, v), paged_cache.load_fp4(cache, table, lens, 8000, 128, dtype=dtype)):
        x, y = x.double().unflatten(-1, (4, 32)), y.double().unflatten(-1, (4, 32))
        assert bool(((x - y).abs() <= x.abs().amax(-1, keepdim=True) / 3.5).all())
        ratio = float((x - y).square().mean().sqrt() / x.square().mean().sqrt())
        assert ratio < 0.2  # a step of 1/2 to 2 around values of 1/2 to 6, uniformly: below 0.17 of each
    again = cache.clone()
    paged_cache.store_fp4(again, *paged_cache.load_fp4(cache, table, lens, 8000, 128, dtype=dtype), table, lens)
    for a, b in zip(paged_cache.load_fp4(again, table, lens, 8000, 128), paged_cache.load_fp4(cache, table, lens, 8000, 128)):
        assert torch.equal(a, b)  # what is held is held exactly


def test_forks_of_many_rows(cuda):
    """Tables and caches past what one block plans."""
    from sfu_repro import paged_cache

    g = torch.Generator().manual_seed(4)
    rows, entries, size, pages = 600, 40, 16, 30000
    lens = torch.randint(0, entries * size + 1, (rows,), generator=g).to(torch.int32)
    order, at = torch.randperm(pages, generator=g).to(torch.int32), 0
    table = torch.full((rows, entries), -1, dtype=torch.int32)
    for i, n in enumerate(lens.tolist()):
        m = -(-n // size)
        table[i, :m] = order[at: at + m]
        at += m
    cache = torch.randint(0, 256, (pages, 32), generator=g, dtype=torch.uint8)
    parents = torch.randint(-1, rows, (900,), generator=g).to(torch.int32)
    for tokens in (0, 40):
        on = cache.to(cuda)
        got = paged_cache.fork_pages([on], table.to(cuda), lens.to(cuda), parents.to(cuda), tokens=tokens, page_size=size)
        out, n, short, moves = ref.fork(table, lens, parents, tokens, size, pages)
        assert torch.equal(got[0].cpu(), out) and torch.equal(got[1].cpu(), n) and got[2].tolist() == [short]
        want = cache.clone()
        for s, d in moves:
            want[d] = cache[s]
        ref.same(on, want)
        packed, used = paged_cache.compact_pages([on], got[0])
        out2, count, moves = ref.compact(out, pages)
        assert torch.equal(packed.cpu(), out2) and used.tolist() == [count]
        after = want.clone()
        for s, d in moves:
            after[d] = want[s]
        ref.same(on, after)
