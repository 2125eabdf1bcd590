"""Attention over a shared prefix with values at the ends of what the operands hold,
against its definition."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _operands(case, cuda, seed=0, scale=1.0):
    dtype, b, t, p, length, hq, hkv, d = case
    g = torch.Generator(device=cuda).manual_seed(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=cuda).to(dt)

    lens = [length - (length - t) * i // b for i in range(b)]
    return [(normal(b, t, hq, d) * scale).to(dt), normal(p, hkv, d), normal(p, hkv, d), normal(b, length, hkv, d),
            normal(b, length, hkv, d), torch.tensor(lens, dtype=torch.int32, device=cuda)]


# dtype, batch, tokens, prefix, suffix, hq, hkv, dim: up to 32 rows a KV head (and a
# cache), up to 64, and more
ROWS = [("bf16", 2, 1, 300, 200, 8, 2, 128), ("f16", 3, 1, 2000, 333, 8, 1, 64), ("bf16", 1, 1, 5000, 100, 4, 4, 64),
        ("f16", 10, 1, 700, 150, 8, 2, 128), ("bf16", 40, 1, 500, 70, 4, 1, 64), ("f16", 40, 1, 900, 70, 8, 2, 128),
        ("bf16", 2, 35, 300, 200, 4, 2, 128), ("f16", 2, 70, 700, 300, 4, 2, 64)]


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("case", ROWS, ids=lambda c: "-".join(map(str, c)))
def test_infinities_that_tokens_see(cuda, case, cap):
    """A sum with an infinity among its values is that infinity, however small its
    probability (down to 2^-90 here); with one of each sign, or a NaN, a NaN.  Wherever the
    keys lie, and for every number of rows.  The other elements keep their bits."""
    from sfu_repro import fa4_runtime

    # scores of up to +- 80 in base 2, which FP16 probabilities do not reach
    t = _operands(case, cuda, scale=6.0 if cap == 0 else 20.0)
    q, pk, pv, sk, sv, lens = t
    b, tokens, hq, d = q.shape
    g = torch.Generator().manual_seed(1)
    bad_p, bad_s = torch.zeros_like(pv), torch.zeros_like(sv)
    kinds = torch.tensor([math.inf, -math.inf, math.nan], dtype=q.dtype)
    # elements 0 .. d/2 in the prefix, d/4 .. 3d/4 in the caches: some in both
    for bad, dims in ((bad_p, range(0, d // 2)), (bad_s.flatten(0, 1), range(d // 4, 3 * d // 4))):
        for e in dims:
            key = torch.randint(0, bad.shape[0], (1,), generator=g).item()
            head = torch.randint(0, bad.shape[1], (1,), generator=g).item()
            bad[key, head, e] = kinds[torch.randint(0, 3, (1,), generator=g).item()]
    pv.masked_fill_(~bad_p.isfinite(), 0)
    sv.masked_fill_(~bad_s.isfinite(), 0)
    clean = fa4_runtime.flash_attn_shared_prefix(*t, softcap=cap)
    assert bool(clean[0].isfinite().all())
    got = fa4_runtime.flash_attn_shared_prefix(q, pk, pv + bad_p, sk, sv + bad_s, lens, softcap=cap)
    # what is not finite: the sum of what each token sees
    want = clean[0].clone()
    group = hq // pk.shape[1]
    seen_p = bad_p.float().sum(0)                                                  # [hkv, d]
    for i in range(b):
        for j in range(tokens):
            n = max(0, int(lens[i]) - tokens + j + 1)
            special = (seen_p + bad_s[i, :n].float().sum(0)).repeat_interleave(group, 0)
            want[i, j] = torch.where(special.isfinite(), want[i, j], special.to(q.dtype))
    assert not bool(want.isfinite().all())
    assert torch.equal(got[1], clean[1])
    assert torch.equal(got[0].isnan(), want.isnan())
    assert torch.equal(got[0].nan_to_num(7.0), want.nan_to_num(7.0))
