"""The definition of attention over a shared prefix in 64 bits, on the operands' device, for
the GPU tests."""

import math

import torch


def definition(q, pk, pv, sk, sv, lens, scale, cap=0.0):
    """out, sum p |v| and sum |v| [B, T, Hq, D], lse [B, Hq, T], in 64 bits."""
    b, t, hq, d = q.shape
    out, size, total = (torch.zeros(b, t, hq, d, dtype=torch.float64, device=q.device) for _ in range(3))
    lse = torch.zeros(b, hq, t, dtype=torch.float64, device=q.device)
    group, own = hq // pk.shape[1], torch.arange(sk.shape[1], device=q.device)
    for i in range(b):
        hidden = own[None] > (int(lens[i]) - t + torch.arange(t, device=q.device))[:, None]         # [t, own]
        hidden = torch.cat([torch.zeros(t, pk.shape[0], dtype=torch.bool, device=q.device), hidden], 1)
        for h in range(hq):
            k, v = (torch.cat([x[:, h // group], y[i, :, h // group]]).double() for x, y in ((pk, sk), (pv, sv)))
            s = q[i, :, h].double() @ k.t().contiguous() * scale
            s = (cap * torch.tanh(s / cap) if cap else s).masked_fill(hidden, -math.inf)
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - s.amax(-1, keepdim=True))  # z may be too large to hold the sum
            p = (p / p.sum(-1, keepdim=True)).masked_fill(hidden, 0)  # also where nothing is seen
            out[i, :, h], size[i, :, h], total[i, :, h], lse[i, h] = p @ v, p @ v.abs(), (~hidden).double() @ v.abs(), z
    return out, size, total, lse
