"""Head norm and rotations at sizes of training, forward and backward, against the formulas in
64 bits: blocks that take several items, heads that fill their splits, results that leave
past the caches.

Tolerances: those of the small sizes (a result is rounded once, off by half a step; ahead of
it 2e-6 of |u_a| + |u_b| of its pair, a gradient 4e-6 of r (|w g| + |n| mean |w g n|)).  A
weight's gradient is added along chains of at most 3 items of 12 heads, 128 rows of a block, 32
partial rows of a thread and 64 threads: 260 additions, within 260 2^-24 + 2e-6 of sum |g n|."""

import pytest
import torch

import qk_rope_reference as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _half_step(t, dtype):
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def _off(got, want, tol):
    ratio = ((got.double() - want).abs() / tol).max()
    assert bool(ratio <= 1), float(ratio)


# dtype, batch, seq, hq, hk, dim, rotary, interleaved, weights: more items than blocks
# (2048) with splits that do not divide a side's blocks, 9 to 12 heads to a split, tokens
# that do not fill the last block's rows, results of less than 32 MiB and of more
NORM = [
    ("bf16", 3, 4099, 24, 9, 128, 128, True, "same"),
    ("f16", 5, 3001, 40, 8, 64, 64, False, "f32"),
    ("f16", 3, 3001, 16, 16, 80, 40, False, "same"),
    ("bf16", 1, 10007, 1, 1, 256, 256, False, "f32"),
    ("f16", 7, 2503, 11, 2, 72, 24, True, "none"),
    ("bf16", 2, 2047, 12, 3, 128, 64, False, "same"),
    ("f16", 2, 4201, 25, 8, 64, 64, True, "f32"),
]


@pytest.mark.parametrize("case", NORM, ids=lambda c: "-".join(map(str, c)))
def test_norm_rope(cuda, case):
    from sfu_repro import rope

    dtype, b, s, hq, hk, d, r, inter, weights = case
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    g = torch.Generator(device=cuda).manual_seed(s)
    # packed, as a projection leaves it; at 64 elements a head, 8 bytes off the widest accesses
    qkv = torch.empty(b * s * (hq + 2 * hk) * d + 4, dtype=dt, device=cuda)[4 if d == 64 else 0:]
    qkv = qkv[: b * s * (hq + 2 * hk) * d].view(b, s, -1).copy_(
        torch.randn(b, s, (hq + 2 * hk) * d, generator=g, device=cuda))
    q, k = qkv[..., : hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d: (hq + hk) * d].unflatten(-1, (hk, d))
    wt = torch.float32 if weights == "f32" else dt
    w = [None if weights == "none" else (1 + 0.3 * torch.randn(d, generator=g, device=cuda)).to(wt) for _ in range(2)]
    dy = [torch.randn(b, h, s, d, generator=g, device=cuda).to(dt) for h in (hq, hk)]
    pos = torch.randint(0, 2 ** 40, (b, s), generator=g, device=cuda)
    inc = rope.phase_increments(r, 500000.0).to(cuda)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, *w) if t is not None]
    wl = leaves[2:] or [None, None]
    out = rope.qk_norm_rope(leaves[0], leaves[1], *wl, inc, pos, eps=EPS, interleaved=inter)
    grads = torch.autograd.grad(out, leaves, dy)
    theta = ref.angles(inc, pos, None, b, s)
    for i, x in enumerate((q, k)):
        x, weight = x.double(), None if w[i] is None else w[i].double()
        tol = _half_step(ref.heads_out(x, weight, theta, EPS, inter, True), dt)
        tol += 2e-6 * ref.pair_size(x, weight, theta, EPS, inter, True)
        _off(out[i].detach(), ref.heads_out(x, weight, theta, EPS, inter, True), tol)
        del tol
        back = dy[i].double().transpose(1, 2)
        gt = ref.rotate(back, -theta, inter)
        pair = ref.pair_size(back, None, theta, EPS, inter, False).transpose(1, 2)
        rstd = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * rstd
        wg = gt if weight is None else gt * weight
        want = rstd * (wg - n * (wg * n).mean(-1, keepdim=True))
        wp = pair if weight is None else pair * weight.abs()
        scale = rstd * (wp + n.abs() * (wp * n.abs()).mean(-1, keepdim=True))
        _off(grads[i], want, _half_step(want, dt) + 4e-6 * scale)
        if weight is not None:
            dw = (gt * n).sum((0, 1, 2))
            tol = (260 * 2.0 ** -24 + 2e-6) * (pair * n.abs()).sum((0, 1, 2)) + _half_step(dw, wt)
            _off(grads[2 + i], dw, tol)


# dtype, batch, seq, hq, hk, dim, rotary, interleaved, axes
AXES = [("bf16", 2, 5003, 32, 8, 128, 128, True, 3), ("f16", 1, 9001, 20, 20, 80, 80, False, 2),
        ("f16", 2, 4001, 17, 17, 96, 48, False, 3), ("bf16", 3, 2001, 9, 3, 64, 64, False, 2)]


@pytest.mark.parametrize("case", AXES, ids=lambda c: "-".join(map(str, c)))
def test_axes(cuda, case):
    from sfu_repro import rope

    dtype, b, s, hq, hk, d, r, inter, n = case
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    g = torch.Generator(device=cuda).manual_seed(s)
    x = [torch.randn(b, s, h, d, generator=g, device=cuda).to(dt).requires_grad_(True) for h in (hq, hk)]
    dy = [torch.randn(b, h, s, d, generator=g, device=cuda).to(dt) for h in (hq, hk)]
    pos = torch.randint(0, 100000, (n, b, s), generator=g, device=cuda)
    axes, inc = (torch.arange(r // 2, device=cuda) % n).to(torch.int32), rope.phase_increments(r, 10000.0).to(cuda)
    out = rope.rope_axes(*x, inc, pos, axes, interleaved=inter)
    grads = torch.autograd.grad(out, x, dy)
    theta = ref.angles(inc, pos, axes, b, s)
    for got, grad, t, d_out in zip(out, grads, x, dy):
        t, back = t.detach().double(), d_out.double().transpose(1, 2)
        want = ref.heads_out(t, None, theta, EPS, inter, False)
        _off(got.detach(), want, _half_step(want, dt) + 2e-6 * ref.pair_size(t, None, theta, EPS, inter, False))
        want = ref.rotate(back, -theta, inter)
        pair = ref.pair_size(back, None, theta, EPS, inter, False).transpose(1, 2)
        _off(grad, want, _half_step(want, dt) + 2e-6 * pair)
