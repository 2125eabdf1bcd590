"""The head norm with its rotation and the rotation by several axes, forward and
backward, against their definitions in 64 bits.

Tolerances.  Results are computed in FP32 and rounded once, off by at most half
a step (eps / 2 of the value; half the smallest subnormal below the normal
range).  Ahead of that rounding a result's FP32 error scales with the pair that
it is made of: sine and cosine are within 9e-8, and the mean, the reciprocal
root, the two products of the norm and the three steps of the rotation add at
most ten roundings of 2^-24 (the mean's tree is seven to eight deep and enters
with half its weight): 2e-6 of |u_a| + |u_b| covers them.  A gradient has a
second mean over the head behind them: 4e-6 of r (|w g| + |n| mean |w g n|).
A weight's gradient adds N rows in FP32 along chains of at most N / 16 + 256
additions, so it is within (N / 16 + 256) 2^-24 + 2e-6 of sum |g n|."""

import math

import pytest
import torch

import qk_rope_reference as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _half_step(t, dtype):
    """Half a step of the type at t, and half its smallest subnormal."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def _increments(rotary, theta=500000.0):
    from sfu_repro import rope

    return rope.phase_increments(rotary, theta)


# dtype, batch, seq, hq, hk, dim, rotary, interleaved, weights, positions, packed
CASES = [
    ("bf16", 1, 1, 1, 1, 8, 8, True, "same", "none", False),
    ("bf16", 2, 3, 3, 1, 16, 16, False, "f32", "seq", False),
    ("f16", 1, 7, 5, 5, 24, 8, False, "same", "batch", True),
    ("f16", 3, 17, 9, 3, 64, 64, True, "same", "batch", True),
    ("bf16", 2, 33, 8, 2, 64, 32, False, "none", "none", True),
    ("f16", 2, 65, 16, 16, 72, 72, False, "f32", "batch", True),
    ("bf16", 3, 50, 12, 4, 80, 40, True, "same", "batch", False),
    ("f16", 1, 100, 4, 4, 96, 48, False, "f32", "far", True),
    ("bf16", 8, 1, 32, 8, 128, 128, False, "same", "far", True),
    ("bf16", 2, 131, 32, 8, 128, 128, True, "f32", "negative", True),
    ("f16", 1, 257, 17, 1, 128, 64, True, "same", "int32", False),
    ("bf16", 1, 40, 8, 8, 256, 256, False, "same", "batch", True),
    ("f16", 2, 31, 3, 2, 256, 8, True, "none", "batch", False),
    ("bf16", 2, 9, 4, 2, 64, 0, True, "same", "none", False),
    ("f16", 5, 700, 8, 8, 40, 40, False, "same", "batch", True),
    ("bf16", 3, 5, 2, 1, 248, 248, True, "f32", "seq", True),
]


def _make(case, seed=0):
    dtype, b, s, hq, hk, d, r, inter, weights, where, packed = case
    g = torch.Generator().manual_seed(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    x = torch.randn(b, s, (hq + 2 * hk) * d, generator=g).to(dt)
    x[0, 0, :d] = 0  # a head of zeros: eps alone under the root
    dq, dk = (torch.randn(b, h, s, d, generator=g).to(dt) for h in (hq, hk))
    wt = torch.float32 if weights == "f32" else dt
    w = [None if weights == "none" else (1 + 0.3 * torch.randn(d, generator=g)).to(wt) for _ in range(2)]
    pos = {"none": None, "seq": torch.arange(5, 5 + s), "batch": torch.randint(0, 10000, (b, s), generator=g),
           "far": torch.randint(0, 2 ** 40, (b, s), generator=g),
           "negative": torch.randint(-2 ** 31, 2 ** 31, (b, s), generator=g),
           "int32": torch.randint(0, 2 ** 31, (b, s), generator=g, dtype=torch.int32)}[where]
    return dt, x, dq, dk, w, pos


def _views(x, case):
    _, b, s, hq, hk, d = case[:6]
    q = x[..., : hq * d].unflatten(-1, (hq, d))
    k = x[..., hq * d: (hq + hk) * d].unflatten(-1, (hk, d))
    return (q, k) if case[10] else (q.contiguous(), k.contiguous())


def _check_out(got, x, w, theta, inter, with_norm, dt):
    want = ref.heads_out(x, w, theta, EPS, inter, with_norm)
    tol = _half_step(want, dt) + 2e-6 * ref.pair_size(x, w, theta, EPS, inter, with_norm)
    off = (got.cpu().double() - want).abs()
    assert got.dtype == dt and got.is_contiguous()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_norm_rope(cuda, case):
    from sfu_repro import rope

    dt, x, dq, dk, w, pos = _make(case)
    _, b, s, hq, hk, d, r, inter = case[:8]
    inc = _increments(r)
    xd = x.to(cuda)
    q, k = _views(xd, case)
    wd = [None if t is None else t.to(cuda) for t in w]
    posd = None if pos is None else pos.to(cuda)
    q_out, k_out = rope.qk_norm_rope(q, k, *wd, inc.to(cuda), posd, eps=EPS, interleaved=inter)
    theta = ref.angles(inc, pos, None, b, s)
    for got, t, weight in ((q_out, _views(x, case)[0], w[0]), (k_out, _views(x, case)[1], w[1])):
        _check_out(got, t.double(), None if weight is None else weight.double(), theta, inter, True, dt)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_norm_rope_gradients(cuda, case):
    from sfu_repro import rope

    dt, x, dq, dk, w, pos = _make(case, seed=1)
    _, b, s, hq, hk, d, r, inter = case[:8]
    inc = _increments(r)
    leaves = [t.detach().requires_grad_(True) for t in _views(x.to(cuda), case)]
    leaves += [t.to(cuda).requires_grad_(True) for t in w if t is not None]
    wd = leaves[2:] if len(leaves) > 2 else [None, None]
    out = rope.qk_norm_rope(leaves[0], leaves[1], *wd, inc.to(cuda), None if pos is None else pos.to(cuda), eps=EPS,
                            interleaved=inter)
    grads = torch.autograd.grad(out, leaves, [dq.to(cuda), dk.to(cuda)])
    theta = ref.angles(inc, pos, None, b, s)
    for i, (t, weight, dy) in enumerate(zip(_views(x, case), w, (dq, dk))):
        t = t.double().requires_grad_(True)
        weight = None if weight is None else weight.double().requires_grad_(True)
        y = ref.heads_out(t, weight, theta, EPS, inter, True)
        want = torch.autograd.grad(y, [t] + ([] if weight is None else [weight]), dy.double())
        with torch.no_grad():
            f = t.detach()
            rstd = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS)
            n = f * rstd
            g = ref.rotate(dy.double().transpose(1, 2), -theta, inter)
            pair = ref.pair_size(dy.double().transpose(1, 2), None, theta, EPS, inter, False).transpose(1, 2)
            wa = 1.0 if weight is None else weight.detach().abs()
            scale = rstd * (wa * pair + n.abs() * (wa * pair * n.abs()).mean(-1, keepdim=True))
            tol = _half_step(want[0], dt) + 4e-6 * scale
            off = (grads[i].cpu().double() - want[0]).abs()
            assert grads[i].dtype == dt
            assert bool((off <= tol).all()), float((off / tol).max())
            if weight is not None:
                rows = b * s * t.shape[2]
                tol = ((rows / 16 + 256) * 2.0 ** -24 + 2e-6) * (pair * n.abs()).sum((0, 1, 2))
                tol = tol + _half_step(want[1], w[i].dtype)
                off = (grads[2 + i].cpu().double() - want[1]).abs()
                assert grads[2 + i].dtype == w[i].dtype
                assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("inter", [True, False])
def test_gradients_against_differences(cuda, inter):
    """The kernel's gradients along random directions, against central
    differences of the 64-bit forward: h^2 / 6 of the third derivative is below
    1e-7 of the sums here, and the FP16 gradients are off by half a step each."""
    from sfu_repro import rope

    case = ("f16", 2, 6, 3, 2, 32, 16, inter, "f32", "batch", False)
    dt, x, dq, dk, w, pos = _make(case, seed=3)
    x[0, 0, :32] = 1  # differences of a head of zeros see eps alone
    inc = _increments(16)
    q, k = _views(x, case)
    leaves = [t.to(cuda).requires_grad_(True) for t in (q, k, *w)]
    out = rope.qk_norm_rope(*leaves, inc.to(cuda), pos.to(cuda), eps=EPS, interleaved=inter)
    grads = [g.cpu().double() for g in torch.autograd.grad(out, leaves, [dq.to(cuda), dk.to(cuda)])]
    theta = ref.angles(inc, pos, None, 2, 6)
    base = [t.double() for t in (q, k, *w)]

    def loss(p):
        return sum((ref.heads_out(p[i], p[2 + i], theta, EPS, inter, True) * dy.double()).sum()
                   for i, dy in enumerate((dq, dk)))

    g = torch.Generator().manual_seed(5)
    for i in range(4):
        v = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        h = 1e-4
        moved = [[t + sign * h * v if j == i else t for j, t in enumerate(base)] for sign in (1, -1)]
        slope = float(loss(moved[0]) - loss(moved[1])) / (2 * h)
        got = float((grads[i] * v).sum())
        steps = float(((grads[i].abs() * torch.finfo(torch.float16).eps / 2 + 1e-4 * 2.0 ** -11) * v.abs()).sum())
        assert abs(got - slope) <= steps + 1e-6 * float((grads[i] * v).abs().sum()) + 1e-6


# dtype, batch, seq, hq, hk, dim, rotary, interleaved, axes, pattern
AXES = [
    ("bf16", 1, 1, 2, 1, 8, 8, True, 2, "sections"),
    ("f16", 2, 40, 4, 4, 80, 80, False, 2, "sections"),
    ("bf16", 2, 33, 8, 2, 128, 128, True, 3, "cyclic"),
    ("bf16", 16, 1, 32, 8, 128, 128, False, 3, "sections"),
    ("f16", 1, 77, 3, 3, 72, 40, False, 3, "cyclic"),
    ("bf16", 1, 130, 9, 1, 256, 128, True, 4, "random"),
    ("f16", 3, 21, 6, 2, 64, 64, True, 1, "sections"),
]


@pytest.mark.parametrize("case", AXES, ids=lambda c: "-".join(map(str, c)))
def test_axes(cuda, case):
    from sfu_repro import rope

    dtype, b, s, hq, hk, d, r, inter, n, pattern = case
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    g = torch.Generator().manual_seed(11)
    q, k = (torch.randn(b, s, h, d, generator=g).to(dt) for h in (hq, hk))
    dq, dk = (torch.randn(b, h, s, d, generator=g).to(dt) for h in (hq, hk))
    pos = torch.randint(-1000, 100000, (n, b, s), generator=g)
    f = r // 2
    axes = {"sections": torch.arange(f) * n // f, "cyclic": torch.arange(f) % n,
            # values past the axes are held to them
            "random": torch.randint(-2, n + 2, (f,), generator=g)}[pattern].to(torch.int32)
    inc = _increments(r, 10000.0)
    qd, kd = (t.to(cuda).requires_grad_(True) for t in (q, k))
    out = rope.rope_axes(qd, kd, inc.to(cuda), pos.to(cuda), axes.to(cuda), interleaved=inter)
    grads = torch.autograd.grad(out, [qd, kd], [dq.to(cuda), dk.to(cuda)])
    theta = ref.angles(inc, pos, axes, b, s)
    for got, grad, t, dy in zip(out, grads, (q, k), (dq, dk)):
        _check_out(got.detach(), t.double(), None, theta, inter, False, dt)
        back = dy.double().transpose(1, 2)
        want = ref.rotate(back, -theta, inter)
        pair = ref.pair_size(back, None, theta, EPS, inter, False).transpose(1, 2)
        off = (grad.cpu().double() - want).abs()
        assert grad.is_contiguous()
        assert bool((off <= _half_step(want, dt) + 2e-6 * pair).all())


def test_norm_with_axes(cuda):
    from sfu_repro import rope

    g = torch.Generator().manual_seed(2)
    q, k = (torch.randn(2, 19, h, 64, generator=g).to(torch.bfloat16) for h in (4, 2))
    pos = torch.randint(0, 500, (3, 2, 19), generator=g, dtype=torch.int32)
    axes, inc = rope.axis_sections((8, 12, 12)), _increments(64)
    out = rope.qk_norm_rope(q.to(cuda), k.to(cuda), None, None, inc.to(cuda), pos.to(cuda),
                            frequency_axes=axes.to(cuda), eps=EPS)
    theta = ref.angles(inc, pos, axes, 2, 19)
    for got, t in zip(out, (q, k)):
        _check_out(got, t.double(), None, theta, True, True, torch.bfloat16)


def test_rotation_matches_rope_apply(spline_ops, cuda):
    """Interleaved pairs at positions 0..S-1 are the rotation of rope_apply,
    whose sines and cosines are FP16 (within 2^-10)."""
    from sfu_repro import rope

    g = torch.Generator().manual_seed(4)
    q, k = (torch.randn(2, 50, h, 128, generator=g).to(torch.bfloat16).to(cuda) for h in (4, 2))
    inc = _increments(128).to(cuda)
    pos = torch.arange(50, device=cuda).expand(1, 2, 50)
    zero = torch.zeros(64, dtype=torch.int32, device=cuda)
    for got, want in zip(rope.rope_axes(q, k, inc, pos, zero), spline_ops.rope_apply_fixed_half_turn_d5_d6_bf16(q, k, inc)):
        assert float((got.float() - want.float()).abs().max()) <= 5.0 * 2 ** -9 + 5.0 * 2 ** -8


def test_layouts_that_need_a_copy(cuda):
    """Odd addresses and strides, a transposed head dimension, broadcast batches."""
    from sfu_repro import rope

    g = torch.Generator().manual_seed(6)
    q = torch.randn(2, 5, 3, 64, generator=g).to(torch.float16).to(cuda)
    k = torch.randn(2, 5, 1, 64, generator=g).to(torch.float16).to(cuda)
    inc, pos = _increments(64).to(cuda), torch.arange(5, device=cuda).expand(2, 5)
    want = rope.qk_norm_rope(q, k, None, None, inc, pos)
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device=cuda)[1:].view(q.shape).copy_(q)
    wide = torch.empty(2, 5, 3, 67, dtype=q.dtype, device=cuda)[..., 2:66].copy_(q)
    turned = q.transpose(2, 3).contiguous().transpose(2, 3)
    inner = q.transpose(1, 2).contiguous().transpose(1, 2)
    for other in (off, wide, turned, inner):
        got = rope.qk_norm_rope(other, k, None, None, inc, pos)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = q[:1].expand(2, 5, 3, 64)
    got = rope.qk_norm_rope(one, k, None, None, inc, pos)
    assert torch.equal(got[0][0], got[0][1]) and torch.equal(got[0][0], want[0][0])
    # gradients arrive in any layout too
    qr = q.clone().requires_grad_(True)
    out = rope.qk_norm_rope(qr, k, None, None, inc, pos)
    d = torch.randn(2, 5, 3, 64, device=cuda).to(torch.float16)
    a, = torch.autograd.grad(out[0], qr, d.transpose(1, 2), retain_graph=True)
    b, = torch.autograd.grad(out[0], qr, d.transpose(1, 2).contiguous(), retain_graph=True)
    c, = torch.autograd.grad(out[0], qr, d.transpose(1, 2).contiguous().transpose(2, 3).contiguous().transpose(2, 3))
    assert torch.equal(a, b) and torch.equal(a, c)


def test_empty(cuda):
    from sfu_repro import rope

    inc = _increments(64).to(cuda)
    for b, s in ((0, 4), (2, 0)):
        q = torch.empty(b, s, 4, 64, dtype=torch.bfloat16, device=cuda, requires_grad=True)
        w = torch.ones(64, device=cuda, requires_grad=True)
        out = rope.qk_norm_rope(q, q, w, w, inc, torch.zeros(b, s, dtype=torch.int64, device=cuda))
        assert out[0].shape == (b, 4, s, 64)
        dq, dw = torch.autograd.grad(out, [q, w], [torch.empty_like(o) for o in out])
        assert dq.shape == q.shape and not dw.any()


def test_only_one_output_used(cuda):
    """A loss of the queries alone: the keys' gradients are zeros, the queries' unchanged."""
    from sfu_repro import rope

    g = torch.Generator().manual_seed(8)
    q, k = (torch.randn(1, 9, h, 64, generator=g).to(torch.bfloat16).to(cuda).requires_grad_(True) for h in (4, 2))
    w = torch.ones(64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    inc = _increments(64).to(cuda)
    out = rope.qk_norm_rope(q, k, w, w, inc)
    d = torch.randn_like(out[0])
    alone = torch.autograd.grad(out[0], [q, k, w], d, retain_graph=True)
    both = torch.autograd.grad(out, [q, k, w], [d, torch.zeros_like(out[1])])
    assert all(torch.equal(a, b) for a, b in zip(alone, both)) and not alone[1].any()


def test_gradients_repeat_bit_for_bit(cuda):
    from sfu_repro import rope

    g = torch.Generator().manual_seed(9)
    q, k = (torch.randn(4, 999, h, 128, generator=g).to(torch.bfloat16).to(cuda).requires_grad_(True) for h in (32, 8))
    w = [torch.ones(128, device=cuda).requires_grad_(True) for _ in range(2)]
    inc = _increments(128).to(cuda)
    d = None
    first = None
    for _ in range(4):
        out = rope.qk_norm_rope(q, k, *w, inc)
        d = d or [torch.randn_like(o) for o in out]
        grads = torch.autograd.grad(out, [q, k, *w], d)
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(grads, first))


def test_infinities_and_nan_stay_in_their_heads(cuda):
    from sfu_repro import rope

    g = torch.Generator().manual_seed(10)
    q, k = (torch.randn(1, 12, h, 128, generator=g).to(torch.bfloat16).to(cuda) for h in (4, 4))
    inc = _increments(128).to(cuda)
    clean = rope.qk_norm_rope(q, k, None, None, inc)
    q[0, 3, 1, 5], k[0, 7, 2, 9] = math.nan, math.inf
    bad = rope.qk_norm_rope(q, k, None, None, inc)
    for c, b, (h, s) in ((clean[0], bad[0], (1, 3)), (clean[1], bad[1], (2, 7))):
        keep = torch.ones(4, 12, dtype=torch.bool, device=cuda)
        keep[h, s] = False
        assert torch.equal(c[0][keep], b[0][keep]) and not b[0, h, s].isfinite().all()


@pytest.mark.parametrize("rotary", [16, 24, 40])
@pytest.mark.parametrize("inter", [True, False])
def test_infinities_behind_the_rotated_elements(cuda, inter, rotary):
    """What is not turned is copied: an infinity or a NaN there reaches nothing else, and
    one in a pair reaches that pair alone; forward and backward."""
    from sfu_repro import rope

    g = torch.Generator().manual_seed(18)
    q, k = (torch.randn(1, 7, h, 48, generator=g).to(torch.float16).to(cuda) for h in (3, 2))
    pos = torch.randint(0, 9999, (2, 1, 7), generator=g).to(cuda)
    axes, inc = (torch.arange(rotary // 2) % 2).to(torch.int32).to(cuda), _increments(rotary).to(cuda)
    other = 1 if inter else rotary // 2

    def run(q, k):
        q, k = (t.clone().requires_grad_(True) for t in (q, k))
        out = rope.rope_axes(q, k, inc, pos, axes, interleaved=inter)
        # the gradients at the results are the operands' values
        return [*(o.detach().transpose(1, 2) for o in out),
                *torch.autograd.grad(out, [q, k], [t.detach().transpose(1, 2) for t in (q, k)])]

    clean = run(q, k)
    for at, value in ((47, math.inf), (rotary, math.nan), (44, -math.inf)):
        q[0, 2, 1, at] = k[0, 5, 0, at] = value
    q[0, 3, 2, 0] = math.nan
    for i, (c, b) in enumerate(zip(clean, run(q, k))):
        where = torch.zeros(c.shape, dtype=torch.bool, device=cuda)
        t, h = (5, 0) if i % 2 else (2, 1)
        for at in (47, rotary, 44):
            where[0, t, h, at] = True
            assert torch.equal(b[0, t, h, at].nan_to_num(7.0), (q, k)[i % 2][0, t, h, at].nan_to_num(7.0))
        if i % 2 == 0:
            where[0, 3, 2, [0, other]] = True
            assert bool(b[0, 3, 2, [0, other]].isnan().all())
        assert torch.equal(c[~where], b[~where])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_at_any_address(cuda, dtype):
    from sfu_repro import rope

    g = torch.Generator().manual_seed(20)
    q, k = (torch.randn(2, 9, h, 64, generator=g).to(torch.bfloat16).to(cuda) for h in (4, 2))
    w = torch.randn(64, generator=g).to(dtype).to(cuda)
    inc, d = _increments(64).to(cuda), None
    results = []
    for off in (0, 1, 2, 4):
        at = torch.empty(68, dtype=dtype, device=cuda)[off: off + 64].copy_(w).requires_grad_(True)
        out = rope.qk_norm_rope(q, k, at, at, inc, interleaved=False)
        d = d or [torch.randn_like(o) for o in out]
        results.append([*out, *torch.autograd.grad(out, at, d)])
        assert all(torch.equal(a, b) for a, b in zip(results[0], results[-1]))


def test_stream_and_graph(cuda):
    """On a stream of the caller's, and captured forward and backward: replays
    with new inputs equal eager calls bit for bit."""
    from sfu_repro import rope

    g = torch.Generator(device=cuda).manual_seed(12)
    q, k = (torch.randn(2, 70, h, 128, generator=g, device=cuda).to(torch.bfloat16).requires_grad_(True) for h in (8, 2))
    w = [torch.ones(128, device=cuda).requires_grad_(True) for _ in range(2)]
    inc = _increments(128).to(cuda)
    pos = torch.randint(0, 1000, (2, 70), generator=g, device=cuda)
    d = [torch.randn(2, h, 70, 128, generator=g, device=cuda).to(torch.bfloat16) for h in (8, 2)]

    def step():
        out = rope.qk_norm_rope(q, k, *w, inc, pos)
        grads = torch.autograd.grad(out, [q, k, *w], d)
        axes = rope.rope_axes(q.detach(), k.detach(), inc, pos.expand(2, 2, 70), zero)
        return [*(o.detach() for o in out), *grads, *axes]

    zero = torch.zeros(64, dtype=torch.int32, device=cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        side = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(side, step()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=g, device=cuda))
            pos.copy_(torch.randint(0, 1000, pos.shape, generator=g, device=cuda))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_refusals_on_the_device(cuda):
    from sfu_repro import rope

    q = torch.zeros(2, 4, 4, 64, dtype=torch.bfloat16, device=cuda)
    k = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device=cuda)
    inc, pos = _increments(64).to(cuda), torch.zeros(2, 4, dtype=torch.int64, device=cuda)
    ok = dict(q=q, k=k, q_weight=None, k_weight=None, phase_increments=inc, positions=pos)
    rope.qk_norm_rope(**ok)
    three = torch.zeros(3, 2, 4, dtype=torch.int64, device=cuda)
    axes = torch.zeros(32, dtype=torch.int32, device=cuda)
    for change, message in [
        (dict(q=q.float()), "float16 or bfloat16"),
        (dict(k=k.half()), "same dtype"),
        (dict(k=k[:1]), "batch sizes"),
        (dict(k=k[:, :3]), "sequence lengths"),
        (dict(k=k[..., :32]), "head dimensions"),
        (dict(k=k[:, :, :0]), "at least one head"),
        (dict(q=q[..., :60], k=k[..., :60]), "multiple of eight"),
        (dict(q=torch.zeros(1, 1, 1, 264, dtype=torch.float16, device=cuda),
              k=torch.zeros(1, 1, 1, 264, dtype=torch.float16, device=cuda)), "up to 256"),
        (dict(q=q[0]), "must have shape"),
        (dict(phase_increments=inc.long()), "int32"),
        (dict(phase_increments=inc.cpu()), "CUDA tensor"),
        (dict(phase_increments=inc[:30]), "multiple of four"),
        (dict(phase_increments=torch.cat([inc, inc])), "at most head_dim / 2"),
        (dict(positions=pos.float()), "int32 or int64"),
        (dict(positions=pos[:, :3]), "agree"),
        (dict(positions=pos[:1]), "agree"),
        (dict(positions=three), "positions must have shape"),
        (dict(positions=pos, frequency_axes=axes), "positions must have shape"),
        (dict(positions=None, frequency_axes=axes), "needs positions"),
        (dict(positions=three, frequency_axes=axes[:8]), "one axis for each frequency"),
        (dict(positions=three, frequency_axes=axes.long()), "int32"),
        (dict(positions=three[:0], frequency_axes=axes), "at least one axis"),
        (dict(q_weight=torch.ones(32, device=cuda)), "shape"),
        (dict(q_weight=torch.ones(64, device=cuda).double()), "float32 or of q's dtype"),
        (dict(q_weight=torch.ones(64, device=cuda), k_weight=torch.ones(64, device=cuda).bfloat16()), "same dtype"),
        (dict(k_weight=torch.ones(64)), "same CUDA device"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            rope.qk_norm_rope(**{**ok, **change})


def test_second_derivatives_are_refused(cuda):
    """A graph through the gradients raises where it is used, not before."""
    from sfu_repro import rope

    g = torch.Generator().manual_seed(14)
    q, k = (torch.randn(1, 5, h, 64, generator=g).to(torch.float16).to(cuda).requires_grad_(True) for h in (4, 2))
    inc, pos = _increments(64).to(cuda), torch.arange(5, device=cuda).expand(1, 1, 5)
    zero = torch.zeros(32, dtype=torch.int32, device=cuda)
    for out, name in ((rope.qk_norm_rope(q, k, None, None, inc), "qk_norm_rope"),
                      (rope.rope_axes(q, k, inc, pos, zero), "rope_axes")):
        d = [torch.ones_like(o).requires_grad_(True) for o in out]
        want = torch.autograd.grad(out, [q, k], d, retain_graph=True)
        for use in (lambda x: x.backward(), lambda x: torch.autograd.grad(x, d[0])):
            grads = torch.autograd.grad(out, [q, k], d, create_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(grads, want))
            with pytest.raises(RuntimeError, match=f"{name} has no second derivative"):
                use(grads[0].sum())
    grads = torch.autograd.grad(rope.qk_norm_rope(q, k, None, None, inc)[0].sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(grads[0].sum(), q)


def test_saved_operands_may_not_change(cuda):
    """An operand edited between forward and backward is refused, as elsewhere in autograd."""
    from sfu_repro import rope

    q = torch.randn(1, 5, 4, 64, device=cuda).half().requires_grad_(True)
    k = torch.randn(1, 5, 4, 64, device=cuda).half()
    pos = torch.arange(5, device=cuda)[None].contiguous()
    out = rope.qk_norm_rope(q, k, None, None, _increments(64).to(cuda), pos)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out[0].sum().backward()


def test_capture_beside_a_living_eager_graph(cuda):
    """A backward pass captured while an eager graph of the same leaves is alive is
    refused (its accumulation nodes belong to the eager stream, which the capture
    may not touch); without that graph it is captured."""
    from sfu_repro import rope

    g = torch.Generator(device=cuda).manual_seed(16)
    q, k = (torch.randn(2, 30, h, 64, generator=g, device=cuda).half().requires_grad_(True) for h in (4, 2))
    w = torch.ones(64, device=cuda).requires_grad_(True)
    inc = _increments(64).to(cuda)
    d = [torch.randn(2, h, 30, 64, generator=g, device=cuda).half() for h in (4, 2)]
    alive = rope.qk_norm_rope(q, k, w, w, inc)
    want = torch.autograd.grad(alive, [q, k, w], d, retain_graph=True)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="an eager graph of the same leaves is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            out = rope.qk_norm_rope(q, k, w, w, inc)
            torch.autograd.grad(out, [q, k, w], d)
    del out, alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope.qk_norm_rope(q, k, w, w, inc)
        held = torch.autograd.grad(out, [q, k, w], d)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
