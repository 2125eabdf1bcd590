"""Attention over a shared prefix at sizes whose blocks take many tiles, against its definition
in 64 bits.

Tolerances.  P and the result are each rounded once (half a step u; in FP16, where
probabilities below the normal range are off by 2^-32 of the largest, as much of sum |v|
over the sum of probabilities relative to the largest, which is at least 1).  A
score's error e is that of D products, D 2^-24 sum |q k| scale, 4e-7 cap with the softcap,
and 1e-5 for the exponent and its instruction.  The sums of O and l take a key at a time at
worst: (keys / 16 + 256) 2^-24 each (sixteen keys a product, then tiles, waves and
parts)."""

import math

import pytest
import torch

from shared_prefix_reference import definition

pytestmark = pytest.mark.gpu


# dtype, batch, tokens, prefix, suffix, hq, hkv, dim, cap, lens ("spread" over the cache, or
# "few" rows of it)
CASES = [
    # 1600 rows a KV head, 128 to a block: 13 tiles and more in a row
    ("bf16", 4, 100, 4099, 700, 32, 8, 128, 0.0, "spread"),
    ("f16", 4, 100, 4099, 700, 32, 8, 64, 0.0, "spread"),
    ("bf16", 4, 100, 4099, 300, 32, 8, 64, 30.0, "spread"),
    ("f16", 3, 133, 4100, 300, 32, 8, 128, 30.0, "spread"),
    # 48 rows, two waves to a row: 12 tiles
    ("bf16", 48, 1, 12001, 90, 32, 32, 128, 0.0, "spread"),
    ("f16", 48, 1, 12001, 90, 32, 32, 64, 0.0, "spread"),
    # caches of many tiles, 128 and 40 rows to a block
    ("bf16", 16, 64, 100, 3001, 32, 8, 128, 0.0, "spread"),
    ("f16", 64, 10, 64, 2001, 16, 4, 64, 0.0, "spread"),
    # K and V beyond 256 MiB, few rows
    ("bf16", 4, 1, 60001, 3001, 16, 8, 128, 0.0, "spread"),
    ("f16", 4, 1, 120001, 3003, 16, 8, 64, 0.0, "spread"),
    # caches allocated for much more than they hold
    ("bf16", 16, 1, 500, 20000, 8, 2, 128, 0.0, "few"),
    ("f16", 5, 3, 0, 50000, 8, 2, 64, 0.0, "few"),
    ("bf16", 3, 40, 200, 9000, 8, 2, 128, 0.0, "few"),
]


@pytest.mark.parametrize("ramp", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_large(cuda, case, ramp):
    """Also with scores that rise and fall by 100 to 140 along the keys (without a cap), so that
    O is rescaled in the middle of the blocks' loops."""
    from sfu_repro import fa4_runtime

    dtype, b, t, p, length, hq, hkv, d, cap, where = case
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    g = torch.Generator(device=cuda).manual_seed(p)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=cuda) * scale

    q = normal(b, t, hq, d, scale=8 if cap else 2)
    pk, pv, sk, sv = normal(p, hkv, d), normal(p, hkv, d).to(dt), normal(b, length, hkv, d), normal(b, length, hkv, d).to(dt)
    if ramp:  # the queries share a direction, along which the keys rise and fall
        q = q + 2
        for k in (pk, sk):
            n = k.shape[-3]
            k.add_((torch.arange(n, device=cuda) * (12.0 / max(n, 1))).sin()[:, None, None] * 3)
    q, pk, sk = q.to(dt), pk.to(dt), sk.to(dt)
    most = length if where == "spread" else length // 20
    lens = torch.tensor([most - (most - min(t, most)) * i // b for i in range(b)], dtype=torch.int32)
    if where == "few":
        lens[b // 2] = 0
    for i in range(b):  # what lies past a sequence is no number
        sk[i, int(lens[i]):], sv[i, int(lens[i]):] = math.nan, math.inf
    lens = lens.to(cuda)
    out, lse = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, sk, sv, lens, softcap=cap)
    scale = 1 / math.sqrt(d)
    live = torch.arange(length, device=cuda)[None, :, None, None] < lens[:, None, None, None]
    sk0, sv0 = (x.masked_fill(~live, 0) for x in (sk, sv))
    want, size, total, want_lse = definition(q, pk, pv, sk0, sv0, lens, scale, cap)
    u = torch.finfo(dt).eps / 2
    keys = p + length
    qk = max([float(x.abs().max()) for x in (pk, sk0) if x.numel()]) * q.double().abs().sum(-1)     # [b, t, hq]
    err = (qk * scale * d * 2.0 ** -24 + 1e-5 + 4e-7 * cap)[..., None]
    chain = (keys / 16 + 256) * 2.0 ** -24
    tol = (u + 2 * err + 2 * chain) * size + u * (1 + u) * want.abs()
    if dtype == "f16":
        tol = tol + 2.0 ** -32 * total + 2.0 ** -25
    off = (out.double() - want).abs()
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool((off <= tol).all()), float((off / tol).max())
    tol_l = err[..., 0].transpose(1, 2) + chain + 1e-6 * want_lse.abs()
    assert bool(((lse.double() - want_lse).abs() <= tol_l)[~empty].all())
