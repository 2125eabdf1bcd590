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
