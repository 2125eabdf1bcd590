"""Attention of a batch over one shared prefix and each sequence's own cache,
against its definition in 64 bits.

Tolerances.  The kernel rounds each probability to the operands' type (half a
step u of it; in FP16 also 2^-25 of what is at least 1 in l, below the normal
range) and the result once more; everything else is FP32.  A score's error d is
that of a sum of D products, at most D 2^-24 sum |q k| scale, with the softcap
4e-7 cap more (its tanh is within 2^-21 of 1), and 1e-5 covers the exponent's
rounding and its instruction.  So an output is within half a step of it plus
(u + 2 (d + 1e-5)) sum p |v|, and lse within d + 1e-5 + 1e-6 |lse|, the sum's
additions among it."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(q, pk, pv, sk, sv, lens, scale, cap):
    """out [B, T, Hq, D], lse [B, Hq, T] in 64 bits, with the tolerances of both."""
    b, t, hq, d = q.shape
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    hkv, cache = pk.shape[1], sk.shape[1]
    out, lse, tol_o, tol_l = (torch.zeros(b, t, hq, n, dtype=torch.float64) for n in (d, 1, d, 1))
    for i in range(b):
        n = min(max(int(lens[i]), 0), cache)
        for h in range(hq):
            k = torch.cat([pk[:, h * hkv // hq], sk[i, :n, h * hkv // hq]]).double()
            v = torch.cat([pv[:, h * hkv // hq], sv[i, :n, h * hkv // hq]]).double()
            for j in range(t):
                c = pk.shape[0] + max(0, n - t + j + 1)
                if c == 0:
                    lse[i, j, h] = -math.inf
                    continue
                x = q[i, j, h].double()
                s = k[:c] @ x * scale
                err = float((k[:c].abs() @ x.abs()).max()) * scale * d * 2.0 ** -24 + 1e-5
                if cap:
                    s = cap * torch.tanh(s / cap)
                    err += 4e-7 * cap
                z = torch.logsumexp(s, 0)
                p = torch.exp(s - z)
                out[i, j, h] = p @ v[:c]
                lse[i, j, h] = z
                tol_o[i, j, h] = ((u + 2 * err) * (p @ v[:c].abs()) + out[i, j, h].abs() * u * (1 + u)
                                  + tiny * (v[:c].abs().sum(0) + 1))
                tol_l[i, j, h] = err + 1e-6 * z.abs()
    return out, lse.squeeze(-1).transpose(1, 2), tol_o, tol_l.squeeze(-1).transpose(1, 2)


# dtype, batch, tokens, prefix, suffix, hq, hkv, dim, cap, lens
CASES = [
    ("bf16", 1, 1, 1, 1, 1, 1, 128, 0.0, [1]),
    ("bf16", 2, 1, 64, 5, 4, 1, 128, 0.0, [5, 1]),
    ("f16", 3, 1, 333, 70, 8, 2, 64, 0.0, [70, 0, 33]),
    ("f16", 2, 1, 1000, 65, 4, 4, 128, 30.0, [64, 65]),
    ("bf16", 5, 1, 4097, 300, 8, 1, 64, 50.0, [300, 1, 2, 299, 128]),
    ("bf16", 9, 1, 515, 40, 16, 4, 128, 0.0, [40, 0, 1, 39, 7, 32, 33, 31, 16]),  # 36 rows: wide prefix, narrow suffix
    ("f16", 2, 7, 100, 50, 10, 2, 64, 0.0, [50, 3]),      # 35 rows a sequence; tokens that see the prefix alone
    ("bf16", 3, 33, 129, 90, 4, 4, 128, 0.0, [90, 33, 34]),
    ("bf16", 1, 150, 257, 150, 2, 1, 128, 30.0, [150]),   # several row tiles of one sequence
    ("f16", 2, 40, 0, 64, 8, 2, 64, 0.0, [64, 40]),       # no prefix
    ("bf16", 2, 3, 0, 10, 4, 2, 128, 0.0, [10, 1]),       # rows that see nothing
    ("bf16", 4, 1, 200, 0, 4, 2, 128, 0.0, [0, 0, 0, 0]),  # no cache
    ("f16", 2, 2, 0, 0, 4, 2, 64, 0.0, [0, 0]),           # no key at all
    ("bf16", 3, 2, 70, 30, 6, 3, 64, 0.0, [-5, 100, 30]),  # lengths held to the cache
    ("bf16", 2, 1, 300, 700, 32, 8, 128, 0.0, [700, 650]),
]


def _make(case, seed=0):
    dtype, b, t, p, length, hq, hkv, d, cap, lens = case
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(b, t, hq, d, generator=g) * (8 if cap else 2)).to(dt)
    pk, pv = (torch.randn(p, hkv, d, generator=g).to(dt) for _ in range(2))
    sk, sv = (torch.randn(b, length, hkv, d, generator=g).to(dt) for _ in range(2))
    for i, n in enumerate(lens):  # what lies past a sequence is no number
        sk[i, max(0, n):], sv[i, max(0, n):] = math.nan, math.inf
    return q, pk, pv, sk, sv, torch.tensor(lens, dtype=torch.int32)


def _check(got, want):
    out, lse, tol_o, tol_l = want
    o, z = got[0].cpu().double(), got[1].cpu().double()
    assert got[1].dtype == torch.float32 and o.shape == out.shape and z.shape == lse.shape
    assert bool(((o - out).abs() <= tol_o).all()), float(((o - out).abs() - tol_o).max())
    empty = lse == -math.inf
    assert torch.equal(z == -math.inf, empty)
    assert bool(((z - lse).abs() <= tol_l)[~empty].all())


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:9])))
def test_shared_prefix(cuda, case):
    from sfu_repro import fa4_runtime

    t = _make(case)
    got = fa4_runtime.flash_attn_shared_prefix(*(x.to(cuda) for x in t), softcap=case[8])
    _check(got, _reference(*t, 1 / math.sqrt(case[7]), case[8]))


def test_scale(cuda):
    from sfu_repro import fa4_runtime

    t = _make(CASES[6], seed=2)
    got = fa4_runtime.flash_attn_shared_prefix(*(x.to(cuda) for x in t), softmax_scale=0.03)
    _check(got, _reference(*t, 0.03, 0.0))


def test_scores_of_any_size(cuda):
    """Scores of several thousand, rising and falling along the keys, so that the
    maximum moves in every part; and all equal."""
    from sfu_repro import fa4_runtime

    q, pk, pv, sk, sv, lens = _make(("bf16", 3, 1, 2000, 64, 4, 2, 128, 0.0, [64, 10, 0]), seed=3)
    ramp = torch.linspace(-8, 8, 2000).sin() * 30
    pk = (pk.float() * 0.1 + ramp[:, None, None]).to(pk.dtype)
    t = (q, pk, pv, sk, sv, lens)
    _check(fa4_runtime.flash_attn_shared_prefix(*(x.to(cuda) for x in t)), _reference(*t, 1 / math.sqrt(128), 0.0))
    t = (q, torch.zeros_like(pk), pv, torch.zeros_like(sk), sv, lens)
    _check(fa4_runtime.flash_attn_shared_prefix(*(x.to(cuda) for x in t)), _reference(*t, 1 / math.sqrt(128), 0.0))


# dtype, tokens, suffix, hq, hkv, dim: up to 32 rows a sequence, up to 64, 128 and more
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("case", [("bf16", 3, 40, 4, 2, 128), ("f16", 5, 33, 4, 1, 64), ("bf16", 25, 70, 4, 2, 64),
                                  ("f16", 30, 64, 2, 1, 128), ("bf16", 100, 130, 2, 2, 128), ("f16", 90, 100, 2, 1, 64)],
                         ids=lambda c: "-".join(map(str, c)))
def test_what_other_tokens_see(cuda, case, cap):
    """A key or value that is no number, ahead of the token that brings it: that
    token and those behind it get what their sums hold, the others the same bits."""
    from sfu_repro import fa4_runtime

    dtype, tokens, suffix, hq, hkv, dim = case
    t = [x.to(cuda) for x in _make((dtype, 2, tokens, 70, suffix, hq, hkv, dim, cap, [suffix, suffix - 2]))]
    q, pk, pv, sk, sv, lens = t
    clean = fa4_runtime.flash_attn_shared_prefix(*t, softcap=cap)
    assert bool(clean[0].isfinite().all())
    h = hkv - 1
    heads = slice(h * hq // hkv, None)
    for b in range(2):
        own = int(lens[b])                      # the last token's row is own - 1
        first, late = tokens - 2, tokens - 1    # tokens that bring what is no number
        sv[b, own - 2, h, 5], sv[b, own - 2, h, 9], sv[b, own - 2, h, dim - 1] = math.inf, -math.inf, math.nan
        sv[b, own - 1, h, 5], sv[b, own - 1, h, 40] = -math.inf, math.inf
    bad = fa4_runtime.flash_attn_shared_prefix(*t, softcap=cap)
    assert torch.equal(bad[1], clean[1])
    want = clean[0].clone()
    want[:, first:, heads, 5], want[:, first:, heads, 9], want[:, first:, heads, dim - 1] = math.inf, -math.inf, math.nan
    want[:, late:, heads, 5], want[:, late:, heads, 40] = math.nan, math.inf
    assert torch.equal(bad[0].isnan(), want.isnan())
    assert torch.equal(bad[0].nan_to_num(7.0), want.nan_to_num(7.0))
    # keys
    sv[~sv.isfinite()] = 0
    clean = fa4_runtime.flash_attn_shared_prefix(*t, softcap=cap)
    for b in range(2):
        sk[b, int(lens[b]) - 1, h] = math.nan
    bad = fa4_runtime.flash_attn_shared_prefix(*t, softcap=cap)
    assert torch.equal(bad[0][:, :late], clean[0][:, :late]) and torch.equal(bad[1][..., :late], clean[1][..., :late])
    assert bool(bad[0][:, late:, heads].isnan().all()) and torch.equal(bad[0][:, late:, :heads.start], clean[0][:, late:, :heads.start])


def test_layouts(cuda):
    """Heads-first caches, a query view of a packed projection, a shared cache row
    behind an expanded batch: the same bits."""
    from sfu_repro import fa4_runtime

    t = [x.to(cuda) for x in _make(("bf16", 3, 2, 90, 40, 8, 2, 128, 0.0, [40, 2, 17]))]
    want = fa4_runtime.flash_attn_shared_prefix(*t)
    q, pk, pv, sk, sv, lens = t
    packed = torch.zeros(3, 2, 24, 128, dtype=q.dtype, device=cuda)
    packed[:, :, 4:12] = q
    other = (packed[:, :, 4:12], *(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (pk, pv)),
             *(x.transpose(1, 2).contiguous().transpose(1, 2) for x in (sk, sv)),
             torch.stack([lens, lens], 1)[:, 0])
    got = fa4_runtime.flash_attn_shared_prefix(*other)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    same = sk[:1].expand(3, -1, -1, -1), sv[:1].expand(3, -1, -1, -1)
    got = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, *same, lens)
    want = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, *(x.contiguous() for x in same), lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits(cuda):
    """Caches whose rows lie 2^28 elements apart, and batches 2^32."""
    from sfu_repro import fa4_runtime

    q, pk, pv, sk, sv, lens = (x.to(cuda) for x in _make(("bf16", 2, 1, 20, 9, 2, 1, 128, 0.0, [9, 4])))
    want = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, sk, sv, lens)
    store = torch.empty(20 * 2 ** 28, dtype=torch.bfloat16, device=cuda)
    far = store.as_strided((20, 1, 128), (2 ** 28, 128, 1)).copy_(pk)
    got = fa4_runtime.flash_attn_shared_prefix(q, far, pv, sk, sv, lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    far_k = store.as_strided((2, 9, 1, 128), (2 ** 32, 2 ** 24, 128, 1)).copy_(sk)
    far_v = store.as_strided((2, 9, 1, 128), (2 ** 32, 2 ** 24, 128, 1), 2 ** 20).copy_(sv)
    got = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, far_k, far_v, lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("program", ["softmax", "softcap", "d4"])
def test_without_prefix_is_causal_attention(spline_ops, cuda, program, dim):
    """Also the D4 softcap, whose scores are the same bits in both kernels."""
    from sfu_repro import fa4_runtime

    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(2, 200, h, dim, generator=g).to(torch.bfloat16).to(cuda) for h in (8, 2, 2))
    q = q * (1 if program == "softmax" else 8)
    args = {"softmax": {}, "softcap": {"softcap": 30.0},
            "d4": {"score_mod": fa4_runtime.create_softcap_scoremod_backend(30.0, 4)}}[program]
    none = torch.empty(0, 2, dim, dtype=torch.bfloat16, device=cuda)
    lens = torch.full((2,), 200, dtype=torch.int32, device=cuda)
    out, lse = fa4_runtime.flash_attn_shared_prefix(q, none, none, k, v, lens, **args)
    want, want_lse = fa4_runtime.flash_attn_fwd(q, k, v, causal=True, **args)
    # both round P and the result to BF16
    assert float((out.float() - want.float()).abs().max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())
    assert float((lse - want_lse).abs().max()) <= 1e-4


@pytest.mark.parametrize("dim", [64, 128])
def test_d4_softcap_decoding(cuda, dim):
    """One token behind a prefix, as the last row of causal attention over the
    whole sequence: the D4 program's scores are the same bits."""
    from sfu_repro import fa4_runtime

    g = torch.Generator().manual_seed(15)
    s, p = 700, 600
    q, k, v = (torch.randn(3, s, h, dim, generator=g).to(torch.bfloat16).to(cuda) for h in (8, 2, 2))
    k, v, q = k.clone(), v.clone(), q * 8
    k[1:, :p], v[1:, :p] = k[:1, :p], v[:1, :p]
    mod = fa4_runtime.create_softcap_scoremod_backend(50.0, 4)
    want, want_lse = fa4_runtime.flash_attn_fwd(q, k, v, causal=True, score_mod=mod)
    for tokens in (1, 40):
        lens = torch.full((3,), s - p, dtype=torch.int32, device=cuda)
        out, lse = fa4_runtime.flash_attn_shared_prefix(q[:, -tokens:], k[0, :p], v[0, :p], k[:, p:], v[:, p:], lens,
                                                        score_mod=mod)
        assert float((out.float() - want[:, -tokens:].float()).abs().max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())
        assert float((lse - want_lse[..., -tokens:]).abs().max()) <= 1e-4


def test_prefix_equals_its_copy_in_every_cache(cuda):
    from sfu_repro import fa4_runtime

    q, pk, pv, sk, sv, lens = (x.to(cuda) for x in _make(("f16", 3, 2, 150, 40, 4, 2, 64, 0.0, [40, 40, 40])))
    out, lse = fa4_runtime.flash_attn_shared_prefix(q, pk, pv, sk, sv, lens)
    whole = [torch.cat([p.expand(3, -1, -1, -1), s], 1) for p, s in ((pk, sk), (pv, sv))]
    other, other_lse = fa4_runtime.flash_attn_shared_prefix(q, pk[:0], pv[:0], *whole, lens + 150)
    assert float((out.float() - other.float()).abs().max()) <= 4 * 2.0 ** -11 * float(pv.float().abs().max())
    assert float((lse - other_lse).abs().max()) <= 1e-4


def test_empty_calls(cuda):
    from sfu_repro import fa4_runtime

    q, pk, pv, sk, sv, lens = (x.to(cuda) for x in _make(CASES[1]))
    out, lse = fa4_runtime.flash_attn_shared_prefix(q[:0], pk, pv, sk[:0], sv[:0], lens[:0])
    assert out.shape == (0, 1, 4, 128) and lse.shape == (0, 4, 1)
    out, lse = fa4_runtime.flash_attn_shared_prefix(q[:, :0], pk, pv, sk, sv, lens)
    assert out.shape == (2, 0, 4, 128) and lse.shape == (2, 4, 0)


def test_repeats_bit_for_bit_and_streams(cuda):
    """The same bits on every call, also where calls on two streams overlap."""
    from sfu_repro import fa4_runtime

    t = [x.to(cuda) for x in _make(("bf16", 33, 1, 3000, 200, 16, 4, 128, 0.0, list(range(33))))]
    u = [x.to(cuda) for x in _make(("bf16", 33, 1, 3000, 200, 16, 4, 128, 0.0, list(range(33, 66))), seed=1)]
    want, want_u = fa4_runtime.flash_attn_shared_prefix(*t), fa4_runtime.flash_attn_shared_prefix(*u)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s, x in zip(streams, (t, u)):
            with torch.cuda.stream(s):
                got.append(fa4_runtime.flash_attn_shared_prefix(*x))
    torch.cuda.synchronize()
    for i, pair in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(pair, (want, want_u)[i % 2]))


def test_graph(cuda):
    """Captured once, replayed as the caches grow: each replay equals an eager call."""
    from sfu_repro import fa4_runtime

    t = [x.to(cuda) for x in _make(("bf16", 4, 1, 700, 90, 8, 2, 128, 0.0, [1, 2, 3, 90]))]
    fa4_runtime.flash_attn_shared_prefix(*t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = fa4_runtime.flash_attn_shared_prefix(*t)
    g = torch.Generator().manual_seed(6)
    t[3].copy_(torch.randn(t[3].shape, generator=g))
    t[4].copy_(torch.randn(t[4].shape, generator=g))
    for step in range(4):
        t[0].copy_(torch.randn(t[0].shape, generator=g))
        t[5].copy_(torch.randint(0, 91, (4,), generator=g))
        graph.replay()
        want = fa4_runtime.flash_attn_shared_prefix(*t)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_decoding_steps(cuda):
    """The operators as a decoding loop uses them: norm and rotation of the new
    token's heads at its own position, its key and value appended to the cache,
    attention over prefix and cache; against the same loop in 64 bits."""
    import qk_rope_reference as ref
    from sfu_repro import fa4_runtime, rope

    b, p, length, hq, hkv, d = 3, 130, 12, 8, 2, 128
    g = torch.Generator().manual_seed(7)
    dt = torch.bfloat16
    inc = rope.phase_increments(d, 500000.0)
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(dt) for _ in range(2)]
    raw_pk, pv = (torch.randn(1, p, hkv, d, generator=g).to(dt) for _ in range(2))
    incd, wd = inc.to(cuda), [x.to(cuda) for x in w]
    _, pk = rope.qk_norm_rope(raw_pk.to(cuda), raw_pk.to(cuda), *wd, incd, interleaved=False)
    pk = pk[0].transpose(0, 1)  # [p, hkv, d], a view
    sk, sv = (torch.full((b, length, hkv, d), math.nan, dtype=dt, device=cuda) for _ in range(2))
    start = torch.tensor([0, 3, 5])
    sk[:, :5], sv[:, :5] = (torch.randn(b, 5, hkv, d, generator=g).to(dt).to(cuda) for _ in range(2))
    for step in range(6):
        qkv = torch.randn(b, 1, hq + 2 * hkv, d, generator=g).to(dt)
        q, k, v = qkv.to(cuda).split((hq, hkv, hkv), 2)
        slot = (start + step).to(cuda)
        q_out, k_out = rope.qk_norm_rope(q, k, *wd, incd, (p + slot)[:, None], interleaved=False)
        rows = torch.arange(b, device=cuda)
        sk[rows, slot], sv[rows, slot] = k_out[:, :, 0], v[:, 0]
        lens = (slot + 1).to(torch.int32)
        got = fa4_runtime.flash_attn_shared_prefix(q_out.transpose(1, 2), pk, pv[0].to(cuda), sk, sv, lens)
        # the kernel's own rotated operands, whose error the rotation's tests bound
        theta = ref.angles(inc, (p + start + step)[:, None], None, b, 1)
        for t, out, weight in ((qkv[:, :, :hq], q_out, w[0]), (qkv[:, :, hq: hq + hkv], k_out, w[1])):
            want = ref.heads_out(t.double(), weight.double(), theta, 1e-6, False, True)
            assert float((out.cpu().double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())
        _check(got, _reference(q_out.transpose(1, 2).cpu(), pk.cpu(), pv[0], sk.cpu(), sv.cpu(), lens.cpu(),
                               1 / math.sqrt(d), 0.0))


def test_refusals_on_the_device(cuda):
    from sfu_repro import fa4_runtime

    names = ("q", "prefix_k", "prefix_v", "suffix_k", "suffix_v", "suffix_lens")
    ok = dict(zip(names, (x.to(cuda) for x in _make(CASES[1]))))
    fa4_runtime.flash_attn_shared_prefix(**ok)
    q, pk, sk = ok["q"], ok["prefix_k"], ok["suffix_k"]
    for change, message in [
        (dict(q=q.float()), "float16 or bfloat16"),
        (dict(q=q[0]), "must have shape"),
        (dict(q=q[..., :96]), "64 or 128"),
        (dict(prefix_k=pk.half()), "q's dtype"),
        (dict(prefix_k=pk[:5]), "same shape"),
        (dict(suffix_v=ok["suffix_v"][:, :3]), "same shape"),
        (dict(prefix_k=pk.cpu()), "CUDA tensor"),
        (dict(q=q[:1]), "batch"),
        (dict(prefix_k=pk.expand(-1, 2, -1), prefix_v=pk.expand(-1, 2, -1)), "kv heads"),
        (dict(q=q[:, :, :0]), "multiple of kv heads"),
        (dict(suffix_lens=ok["suffix_lens"].long()), "suffix_lens"),
        (dict(suffix_lens=ok["suffix_lens"][:1]), "suffix_lens"),
        (dict(suffix_lens=ok["suffix_lens"].cpu()), "suffix_lens"),
        (dict(softmax_scale=0.0), "softmax_scale"),
        (dict(softmax_scale=math.nan), "softmax_scale"),
        (dict(q=torch.empty(q.numel() + 4, dtype=q.dtype, device=cuda)[4:].view(q.shape)), "alignment"),
        (dict(prefix_k=torch.zeros(64, 1, 132, dtype=q.dtype, device=cuda)[..., :128]), "multiples of 8"),
        (dict(suffix_k=sk.transpose(1, 3).contiguous().transpose(1, 3)), "contiguous head dimension"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            fa4_runtime.flash_attn_shared_prefix(**{**ok, **change})
    with pytest.raises(NotImplementedError, match="hardware"):
        fa4_runtime.flash_attn_shared_prefix(**ok, exp2_emu_backend="d3", exp2_emu_freq=4)
    mod = fa4_runtime.create_softcap_scoremod_backend(30.0, 4)
    with pytest.raises(TypeError, match="bfloat16 program"):
        half = {n: t.half() if t.dtype == torch.bfloat16 else t for n, t in ok.items()}
        fa4_runtime.flash_attn_shared_prefix(**half, score_mod=mod)
    with pytest.raises(TypeError, match="unexpected keyword"):
        fa4_runtime.flash_attn_shared_prefix(**ok, causal=True)
    with pytest.raises(RuntimeError, match="no backward"):
        fa4_runtime.flash_attn_shared_prefix(**{**ok, "q": q.clone().requires_grad_(True)})
