"""Attention over 4-bit pages: each score program in each of the kernels that a call's rows choose (one token
with up to 4 rows a KV head and with 5 to 8, up to 16 rows, 32, 64, 128), and the one-token kernels' keys that
are not there or no numbers."""

import math

import pytest
import torch

import paged_reference as ref
from test_gpu_paged_attention import make, run

pytestmark = pytest.mark.gpu

# dtype, batch, tokens, hq, hkv, dim, page_size, cap, lens: softcapped decoding
CASES = [
    ("bf16", 3, 1, 8, 2, 128, 64, 30.0, [700, 1, 256]),
    ("bf16", 2, 1, 16, 2, 128, 16, 50.0, [2000, 257]),
    ("bf16", 2, 1, 5, 1, 128, 32, 20.0, [255, 513]),
    ("bf16", 3, 1, 3, 3, 128, 64, 30.0, [300, 0, 1000]),
    ("bf16", 1, 1, 4, 1, 128, 16, 30.0, [9000]),
    ("bf16", 2, 1, 6, 1, 64, 16, 20.0, [700, 64]),
    ("bf16", 2, 1, 4, 2, 64, 32, 30.0, [1000, 31]),
    ("f16", 2, 1, 8, 1, 64, 64, 50.0, [600, 2]),
    ("f16", 2, 1, 8, 2, 128, 16, 30.0, [300, 513]),
    ("bf16", 2, 6, 8, 2, 128, 64, 30.0, [400, 6]),      # 24 rows
    ("bf16", 1, 12, 4, 1, 64, 16, 20.0, [200]),         # 48
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:8])))
def test_softcap(cuda, case):
    t = make(case, seed=31)
    ref.check(run(t, cuda, softcap=case[7]), ref.attention(*t, 1 / math.sqrt(case[5]), case[7]))


# tokens, hq, hkv, lens
D4 = [(1, 4, 1, [700, 257]), (1, 2, 2, [300, 1]), (1, 8, 1, [513, 64]), (1, 5, 1, [300, 256]), (1, 32, 2, [300, 17]),
      (4, 8, 2, [200, 90]), (7, 4, 1, [200, 7]), (12, 4, 1, [150, 40]), (33, 4, 1, [150, 40]), (70, 4, 2, [400, 70])]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", D4, ids=lambda c: "-".join(map(str, c[:3])))
def test_d4_softcap(cuda, case, dim):
    """The D4 program over what the cache holds, as the shared-prefix attention computes it from the same
    numbers a token at a time.  Queries are whole numbers up to 4 and keys multiples of 1/2 up to 6, so that scores are
    exact in any order of their sums and the programs begin with the same bits.  From there both have P
    in two BF16 terms (2^-16) and sums in FP32 (n 2^-22) of at most the largest value, and each rounds its result
    by half a step, which is eps / 2 = 2^-8 of it (BF16 keeps eight bits): 2^-7 for the two; lse within 1e-5 and n 2^-22."""
    from sfu_repro import fa4_runtime, paged_cache

    tokens, hq, hkv, lens = case
    q, cache, table, n = (x.to(cuda) for x in make(("bf16", 2, tokens, hq, hkv, dim, 16, 0.0, lens), seed=32))
    q = torch.randint(-4, 5, q.shape, generator=torch.Generator().manual_seed(33)).to(q)
    cache[:, 0, :, 16 * dim // 2:] = 127
    mod = fa4_runtime.create_softcap_scoremod_backend(50.0, 4)
    out, lse = fa4_runtime.flash_attn_paged_fp4(q, cache, table, n, softmax_scale=0.25, score_mod=mod)
    for b in range(2):
        k, v = paged_cache.load_fp4(cache, table[b:b + 1], n[b:b + 1], lens[b], dim)
        size = float(v.float().abs().max())
        for t in range(tokens):
            seen = lens[b] - tokens + 1 + t
            kk, vv = k[:, :seen].contiguous(), v[:, :seen].contiguous()
            want, want_lse = fa4_runtime.flash_attn_shared_prefix(q[b:b + 1, t:t + 1], k[0, :0], v[0, :0], kk, vv, n[b:b + 1] * 0 + seen,
                                                                  softmax_scale=0.25, score_mod=mod)
            got, want = out[b:b + 1, t:t + 1].double(), want.double()
            off = (got - want).abs() - want.abs() * 2.0 ** -7 * 1.01 - (2 * 2.0 ** -16 + seen * 2.0 ** -21) * size
            assert float(off.max()) <= 0, (b, t)
            assert float((lse[b, :, t] - want_lse[0, :, 0]).abs().max()) <= 1e-5 + seen * 2.0 ** -22 + 1e-6 * 60  # lse is below 60
    assert bool(lse.isfinite().all())


# dtype, hq, hkv, dim, cap: the one-token kernels
ONE = [("bf16", 4, 1, 64, 0.0), ("f16", 8, 1, 64, 0.0), ("bf16", 8, 2, 128, 30.0), ("bf16", 16, 2, 128, 30.0), ("bf16", 4, 1, 128, 0.0),
       ("f16", 4, 1, 128, 30.0)]


@pytest.mark.parametrize("case", ONE, ids=lambda c: "-".join(map(str, c)))
def test_pages_that_one_token_does_not_find(cuda, case):
    """Entries that name no page, in the middle, at the start, and all along a sequence."""
    dtype, hq, hkv, dim, cap = case
    t = make((dtype, 3, 1, hq, hkv, dim, 16, cap, [900, 290, 70]), seed=34)
    table = t[2]
    table[0, 0], table[0, 20], table[0, 21], table[0, 22], table[1, 18] = -1, 2 ** 31 - 1, t[1].shape[0], -1, -2 ** 31
    table[2] = -1
    ref.check(run(t, cuda, softcap=cap), ref.attention(*t, 1 / math.sqrt(dim), cap))


@pytest.mark.parametrize("case", ONE, ids=lambda c: "-".join(map(str, c)))
def test_blocks_that_are_no_numbers_for_one_token(cuda, case):
    """In a value: its elements of its head's rows; in a key: the rows; behind the keys: nothing."""
    dtype, hq, hkv, dim, cap = case
    t = make((dtype, 3, 1, hq, hkv, dim, 16, cap, [600, 301, 40]), seed=35)
    q, cache, table, lens = t
    codes, row = 16 * dim // 2, dim // 32
    where = lambda b, x: (int(table[b, x // 16]), codes + x % 16 * row)  # noqa: E731
    page, at = where(0, 333)
    cache[page, 1, hkv - 1, at + row - 1] = 255
    page, at = where(1, 300)  # the last key
    cache[page, 1, 0, at] = 254
    page, at = where(2, 5)
    cache[page, 0, hkv - 1, at + 1] = 253
    want = ref.attention(*t, 1 / math.sqrt(dim), cap)
    group = hq // hkv
    assert int(want[0].isnan().sum()) == group * (32 + 32 + dim) and bool(want[0][2, 0, -group:].isnan().all())
    ref.check(run(t, cuda, softcap=cap), want)
