"""Calls of more than 16384 new tokens over a cache in pages of 4-bit numbers."""

import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

TOKENS = 20001


def _cache(device, hkv=2, dim=64, size=64, rows=1):
    from sfu_repro import paged_cache

    entries = -(-TOKENS // size)
    table = torch.randperm(rows * entries, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(rows, entries)
    return paged_cache.fp4_cache(rows * entries, hkv, dim, size, device=device), table.to(device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_store_and_load_of_a_prompt(cuda, dtype):
    """In one call, the same as in two; the second sequence is shorter (padded on the left)."""
    from sfu_repro import paged_cache

    g = torch.Generator(device=cuda).manual_seed(2)
    k, v = (torch.randn(2, TOKENS, 2, 64, generator=g, device=cuda, dtype=dtype) for _ in range(2))
    cache, table = _cache(cuda, rows=2)
    lens = torch.tensor([TOKENS, 17000], dtype=torch.int32, device=cuda)
    paged_cache.store_fp4(cache, k, v, table, lens)
    parts, at = torch.zeros_like(cache), 12345
    paged_cache.store_fp4(parts, k[:, :at], v[:, :at], table, lens - (TOKENS - at))
    paged_cache.store_fp4(parts, k[:, at:], v[:, at:], table, lens)
    assert torch.equal(cache, parts)
    got = paged_cache.load_fp4(cache, table, lens, TOKENS, 64, dtype=dtype)
    for x, y in zip((k, v), got):
        assert not bool(y[1, : TOKENS - 17000].any())
        ref.same(y[0, ::97], ref.nearest(x[0, ::97].cpu()))
        ref.same(y[1, TOKENS - 17000 :: 97], ref.nearest(x[1, TOKENS - 17000 :: 97].cpu()))


def test_attention_of_a_prompt(cuda):
    """Its first, middle and last tokens against the definition."""
    from sfu_repro import fa4_runtime

    g = torch.Generator(device=cuda).manual_seed(3)
    cache, table = _cache(cuda)
    cache.copy_(torch.randint(0, 256, cache.shape, generator=g, device=cuda, dtype=torch.uint8))
    codes = 64 * 32
    cache[..., codes:] = cache[..., codes:] % 4 + 123
    q = torch.randn(1, TOKENS, 4, 64, generator=g, device=cuda).to(torch.bfloat16)
    lens = torch.tensor([TOKENS], dtype=torch.int32, device=cuda)
    out, lse = fa4_runtime.flash_attn_paged_fp4(q, cache, table, lens)
    for at, n in ((0, 100), (16350, 60), (TOKENS - 33, 33)):
        want = ref.attention_at_scale(q[:, at:at + n], cache, table, torch.tensor([at + n]), 1 / 8)
        ref.check((out[:, at:at + n], lse[..., at:at + n]), want)


def test_sizes_are_refused_by_name(cuda):
    from sfu_repro import fa4_runtime, paged_cache

    cache, table = _cache(cuda)
    lens = torch.tensor([TOKENS], dtype=torch.int32, device=cuda)
    kv = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16, device=cuda).expand(1, TOKENS + 100, 2, 64)
    for call in (lambda: paged_cache.store_fp4(cache, kv, kv, table, lens),
                 lambda: paged_cache.load_fp4(cache, table, lens, TOKENS + 100, 64),
                 lambda: fa4_runtime.flash_attn_paged_fp4(kv, cache, table, lens)):
        with pytest.raises(RuntimeError, match="more than 16384 tokens have to fit a row of the table"):
            call()
    short = table[:, :10]
    paged_cache.store_fp4(cache, kv[:, :16384], kv[:, :16384], short, torch.full_like(lens, 640))  # as many as ever
    wide = table.new_zeros(1, 1).expand(1, 2 ** 24 + 1)
    with pytest.raises(RuntimeError, match="2\\^30 keys"):
        paged_cache.load_fp4(cache, wide, lens, 1, 64)
    many = table.new_zeros(1, 1).expand(2 ** 22, 1)
    k = kv[:, :1].expand(2 ** 22, 100, 2, 64)
    with pytest.raises(RuntimeError, match="2\\^34 elements"):
        paged_cache.store_fp4(cache, k, k, many, lens.expand(2 ** 22))
