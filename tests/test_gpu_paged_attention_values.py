"""Attention over a cache in pages of 4-bit numbers: what a call's shape makes no difference to."""

import math

import pytest
import torch

import paged_reference as ref
from test_gpu_paged_attention import make, run

pytestmark = pytest.mark.gpu


def _by_token(t, scale, cap=0.0):
    """paged_reference.attention of each token alone, whose tolerances are those of probabilities in two
    terms: token j of T over lens - T + 1 + j keys."""
    q, cache, table, lens = t
    n = q.shape[1]
    parts = [ref.attention(q[:, j:j + 1], cache, table, lens - n + 1 + j, scale, cap) for j in range(n)]
    return tuple(torch.cat([p[i] for p in parts], 1 if i % 2 == 0 else 2) for i in (0, 2, 1, 3))


# dtype, batch, tokens, hq, hkv, dim, page_size, cap, lens: tiles of 64 and of 128 rows, one and several
@pytest.mark.parametrize("case", [
    ("bf16", 3, 5, 16, 2, 128, 64, 0.0, [700, 3, 64]), ("bf16", 2, 17, 8, 4, 64, 16, 0.0, [300, 17]),
    ("bf16", 2, 33, 4, 1, 128, 16, 0.0, [400, 90]), ("bf16", 1, 70, 4, 2, 64, 32, 20.0, [200]),
    ("f16", 2, 33, 4, 1, 128, 16, 0.0, [400, 90])], ids=lambda c: "-".join(map(str, c[:8])))
def test_many_rows_are_as_exact_as_one_token(cuda, case):
    """More than 32 rows to a KV head, within what a token of its own is held to."""
    t = make(case, seed=21)
    out, tol_o, lse, tol_l = _by_token(t, 1 / math.sqrt(case[5]), case[7])
    ref.check(run(t, cuda, softcap=case[7]), (out, lse, tol_o, tol_l))


# dtype, tokens, hq, hkv, dim: the one-token kernels of 2 and 4 classes, 16 rows, 32, 64 and 128
@pytest.mark.parametrize("case", [("bf16", 1, 4, 1, 64), ("bf16", 1, 8, 1, 64), ("bf16", 1, 4, 2, 128), ("f16", 1, 4, 2, 128),
                                  ("bf16", 6, 8, 2, 64), ("bf16", 9, 4, 1, 128), ("bf16", 70, 2, 1, 64), ("f16", 40, 2, 1, 128)],
                         ids=lambda c: "-".join(map(str, c)))
def test_values_up_to_2_to_the_120_over_the_keys(cuda, case):
    """Scores that rise by 7.9 (log2) behind the first keys, so that the running maximum stays and the
    probabilities behind reach 2^7.9: 600 keys of values up to 6 2^108 (their sum is below 2^120)."""
    dtype, tokens, hq, hkv, dim = case
    size = 64
    q, cache, table, lens = make((dtype, 2, tokens, hq, hkv, dim, size, 0.0, [600, 530]), seed=22)
    codes = size * dim // 2
    q[:] = 0
    q[..., 0] = 1
    cache[:, 0] = 0
    cache[:, 0, :, codes:] = 127
    for b in range(2):
        for x in range(256, int(lens[b])):  # keys of 1 there
            cache[int(table[b, x // size]), 0, :, x % size * dim // 2] = 2
    g = torch.Generator().manual_seed(23)
    cache[:, 1, :, codes:] = torch.randint(100, 127 + 109, cache[:, 1, :, codes:].shape, generator=g, dtype=torch.uint8)
    scale = 7.9 * math.log(2)
    t = (q, cache, table, lens)
    want = ref.attention(*t, scale)
    assert bool(want[0].isfinite().all()) and float(want[0].abs().max()) > 2.0 ** 100
    got = run(t, cuda, softmax_scale=scale)
    far = want[0].abs() + want[2] >= float(torch.finfo(q.dtype).max) * 0.99
    assert bool((got[0].cpu().double().abs() >= float(torch.finfo(q.dtype).max) * 0.97)[far].all())
    off = (got[0].cpu().double() - want[0]).abs() - want[2]
    assert bool((off <= 0)[~far].all())
    assert bool(((got[1].cpu().double() - want[1]).abs() <= want[3]).all())
