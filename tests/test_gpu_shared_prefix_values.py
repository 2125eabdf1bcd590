"""Attention over a shared prefix with values at the ends of what the operands hold,
against its definition."""

import math

import pytest
import torch

from shared_prefix_reference import definition

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


@pytest.mark.parametrize("case", ROWS, ids=lambda c: "-".join(map(str, c)))
def test_scores_of_any_magnitude(cuda, case):
    """Scores of both signs, from 1 to 2^106 (2^30 in FP16), the sizes and signs side
    by side in the rows: each row is the mean over the keys of its largest score, or
    an ordinary softmax.  Keys are whole multiples of one vector, so that scores are exact
    but for the scale.  An output is off by the rounding of P (half a step u of sum p |v|,
    and in FP16 2^-25 of each |v| below the normal range), of itself, and 2e-5 for the
    exponents; lse by 2e-5 and eight roundings of 2^-24."""
    from sfu_repro import fa4_runtime

    q, pk, pv, sk, sv, lens = _operands(case, cuda, seed=3)
    bf = q.dtype == torch.bfloat16
    sizes = [2.0 ** n for n in ((-4, 0, 14, 18, 30, 60, 100) if bf else (-12, -9, 0, 5, 10, 15))]
    step = 1.0 if bf else 512.0
    b, t, hq, d = q.shape
    signed = torch.tensor([sign * x for x in sizes for sign in (1.0, -1.0)], device=cuda)
    rows = torch.arange(b * t * hq, device=cuda).view(b, t, hq) * 5 + 3  # every size meets every row of a tile
    q = signed[rows % len(signed)][..., None].expand(q.shape).to(q.dtype).contiguous()
    for k in (pk, sk):
        g = torch.Generator(device=cuda).manual_seed(k.dim())
        k.copy_((torch.randint(1, 8, k.shape[:-1], generator=g, device=cuda) * step)[..., None].expand(k.shape))
    scale = float(torch.tensor(1 / math.sqrt(d), dtype=torch.float32))
    out, lse = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, sk, sv, lens, softmax_scale=scale)
    want, size, total, want_lse = definition(q, pk, pv, sk, sv, lens, scale)
    u = torch.finfo(q.dtype).eps / 2
    tol = (u + 2e-5) * size + u * (1 + u) * want.abs()
    if not bf:
        tol = tol + 2.0 ** -25 * (total + 1)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).nan_to_num(math.inf).max())
    assert bool(((lse.double() - want_lse).abs() <= 2e-5 + 2.0 ** -21 * want_lse.abs()).all())


def test_a_row_whose_scores_lie_below_all_others(cuda):
    """One key with a score of -1e31: the row is its value."""
    from sfu_repro import fa4_runtime

    for d in (64, 128):
        q = torch.full((2, 1, 4, d), -1e15, dtype=torch.bfloat16, device=cuda)
        k = torch.full((2, 1, 2, d), 1e15, dtype=torch.bfloat16, device=cuda)
        v = torch.randn(2, 1, 2, d, device=cuda).to(torch.bfloat16)
        none = k[0, :0]
        lens = torch.ones(2, dtype=torch.int32, device=cuda)
        out, lse = fa4_runtime.flash_attn_shared_prefix(q, none, none, k, v, lens)
        assert torch.equal(out[:, 0], v[:, 0].repeat_interleave(2, 1)) and bool(lse.isfinite().all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("batch", [1, 12, 33])
def test_many_small_probabilities(cuda, batch, d):
    """FP16: in every 32 keys 31 at 2^-26.5 of one whose value is zero.  Probabilities
    below the normal range are off by 2^-25 in units of at most 2^-7 of the largest, so an
    output by 2^-32 of sum |v| over the largest ones' number."""
    from sfu_repro import fa4_runtime

    q = torch.ones(batch, 1, 4, d, dtype=torch.float16, device=cuda)
    k = torch.full((9600, 1, d), -1.625, dtype=torch.float16, device=cuda)
    v = torch.randint(20000, 60000, (9600, 1, d), device=cuda).to(torch.float16)
    k[5::32], v[5::32] = 0, 0
    none = torch.zeros(batch, 0, 1, d, dtype=torch.float16, device=cuda)
    lens = torch.zeros(batch, dtype=torch.int32, device=cuda)
    scale = 18.375 / (1.625 * d)
    out, _ = fa4_runtime.flash_attn_shared_prefix(q, k, v, none, none, lens, softmax_scale=scale)
    want, size, total, _ = definition(q, k, v, none, none, lens, scale)
    u = 2.0 ** -11
    tol = (u + 2e-5) * size + u * (1 + u) * want + 2.0 ** -32 * total / 300 + 2.0 ** -25
    assert float(want.min()) > 0.01 and float((tol / want).max()) < 0.05
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("batch", [2, 20])
def test_rows_whose_scores_are_all_minus_infinity(cuda, batch):
    """As a row that sees no key: zeros and an lse of -inf; the other rows are untouched."""
    from sfu_repro import fa4_runtime

    q, pk, pv, sk, sv, lens = _operands(("bf16", batch, 1, 90, 40, 4, 2, 128), cuda, seed=5)
    q, pk, sk = q.abs(), pk.abs(), sk.abs()
    clean = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, sk, sv, lens)
    pk[:, 1], sk[:, :, 1] = -math.inf, -math.inf
    out, lse = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, sk, sv, lens)
    assert not bool(out[:, :, 2:].any()) and bool((lse[:, 2:] == -math.inf).all())
    assert torch.equal(out[:, :, :2], clean[0][:, :, :2]) and torch.equal(lse[:, :2], clean[1][:, :2])
