"""The definitions of the head norm and the rotations in 64 bits, on the CPU,
for the GPU tests; elementary operations only, so autograd differentiates them."""

import math

import torch


def angles(increments, positions, axes, batch, seq):
    """[batch, seq, 1, frequencies] in radians; exact modulo a turn."""
    inc = increments.long() % 2 ** 32
    if positions is None:
        positions = torch.arange(seq).expand(batch, seq)
    if axes is not None:
        held = axes.long().clamp(0, positions.shape[0] - 1)
        p = torch.stack([positions[a].long() for a in held.tolist()], -1)
    else:
        p = positions.long().expand(batch, seq)[..., None]
    phase = (p % 2 ** 32) * inc % 2 ** 32 if inc.numel() == 0 else _mulmod(p % 2 ** 32, inc)
    return (phase.double() * (2 * math.pi / 2 ** 32)).unsqueeze(2)


def _mulmod(a, b):
    """a * b modulo 2^32 of values below 2^32, without passing 63 bits."""
    lo, hi = a % 2 ** 16, a // 2 ** 16
    return (lo * b + (hi * b) % 2 ** 16 * 2 ** 16) % 2 ** 32


def rotate(u, theta, interleaved):
    """u [batch, seq, heads, dim] with the leading 2F elements of a head turned."""
    f = theta.shape[-1]
    head, rest = u[..., : 2 * f], u[..., 2 * f:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :f], head[..., f:])
    ra, rb = a * theta.cos() - b * theta.sin(), a * theta.sin() + b * theta.cos()
    head = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((head, rest), -1)


def norm(x, weight, eps):
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return u if weight is None else u * weight


def heads_out(x, weight, theta, eps, interleaved, with_norm):
    """[batch, heads, seq, dim]."""
    u = norm(x, weight, eps) if with_norm else x
    return rotate(u, theta, interleaved).transpose(1, 2)


def pair_size(x, weight, theta, eps, interleaved, with_norm):
    """What an output's error scales with: |u_a| + |u_b| of its pair (|u| where
    nothing turns), [batch, heads, seq, dim]."""
    u = (norm(x, weight, eps) if with_norm else x).abs()
    f = theta.shape[-1]
    head, rest = u[..., : 2 * f], u[..., 2 * f:]
    if interleaved:
        t = head[..., 0::2] + head[..., 1::2]
        head = torch.stack((t, t), -1).flatten(-2)
    else:
        t = head[..., :f] + head[..., f:]
        head = torch.cat((t, t), -1)
    return torch.cat((head, rest), -1).transpose(1, 2)
