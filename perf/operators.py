"""Operators between an attention layer's projections and its output.

Three that serve a model next to the fused attention: the norm of each query and
key head with its rotary rotation in one pass (``qk_norm_rope``), the rotary
rotation by positions of several axes (``rope_axes``), and the attention of a
batch over one prefix that all its sequences share (``shared_prefix``).  The
first two train as well.  ``listed`` holds one size of each use, ``draw`` the
ranges.  ``run`` computes the formulas in elementary operations, or, with
``own``, makes the calls that a user of this package makes.
"""

import math
import os
import sys

import torch

own = False

THETA = 500000.0  # rotary base
EPS = 1e-6        # of the norms
TURN = 2 ** 32    # a phase increment's units per turn


def listed():
    return [
        # A decoding step: eight sequences, one token each, at far positions of
        # their own.  The smallest call: latency and launches.
        {"name": "norm_rope_decode", "op": "qk_norm_rope", "dtype": "bf16", "batch": 8, "seq": 1, "hq": 32, "hkv": 8,
         "hd": 128, "rotary": 128, "interleaved": False, "weight": "same", "packed": True, "train": False},
        # Prefill of a long prompt, Q and K as views of the packed projection.
        {"name": "norm_rope_prefill", "op": "qk_norm_rope", "dtype": "bf16", "batch": 1, "seq": 6001, "hq": 32,
         "hkv": 8, "hd": 128, "rotary": 128, "interleaved": False, "weight": "same", "packed": True, "train": False},
        # A training step's batch, forward and backward, the weights' gradients
        # among it.
        {"name": "norm_rope_train", "op": "qk_norm_rope", "dtype": "bf16", "batch": 4, "seq": 4096, "hq": 32,
         "hkv": 8, "hd": 128, "rotary": 128, "interleaved": True, "weight": "same", "packed": False, "train": True},
        # A ragged FP16 batch, head size 80, half of it rotated, FP32 weights.
        {"name": "norm_rope_odd_train", "op": "qk_norm_rope", "dtype": "f16", "batch": 3, "seq": 1001, "hq": 16,
         "hkv": 16, "hd": 80, "rotary": 40, "interleaved": False, "weight": "f32", "packed": True, "train": True},
        # A decoding step of a model with time, height and width positions.
        {"name": "axes_decode", "op": "rope_axes", "dtype": "bf16", "batch": 16, "seq": 1, "hq": 32, "hkv": 8,
         "hd": 128, "rotary": 128, "axes": 3, "cyclic": False, "interleaved": False, "packed": True, "train": False},
        # A vision encoder: 9000 patches, height and width, FP16, head size 80.
        {"name": "axes_vision", "op": "rope_axes", "dtype": "f16", "batch": 1, "seq": 9000, "hq": 16, "hkv": 16,
         "hd": 80, "rotary": 80, "axes": 2, "cyclic": False, "interleaved": False, "packed": True, "train": False},
        # Training on video: text, then frames, three axes in turn over the
        # frequencies.
        {"name": "axes_video_train", "op": "rope_axes", "dtype": "bf16", "batch": 2, "seq": 8190, "hq": 32, "hkv": 8,
         "hd": 128, "rotary": 128, "axes": 3, "cyclic": True, "interleaved": True, "packed": False, "train": True},
        # Decoding behind a short system prompt: launches and latency.
        {"name": "prefix_decode_small", "op": "shared_prefix", "dtype": "bf16", "batch": 8, "tokens": 1,
         "prefix": 1024, "suffix": 256, "hq": 32, "hkv": 8, "hd": 128, "softcap": 0.0},
        # A large batch that answers from one long document.
        {"name": "prefix_decode_batch", "op": "shared_prefix", "dtype": "bf16", "batch": 64, "tokens": 1,
         "prefix": 32768, "suffix": 2048, "hq": 32, "hkv": 8, "hd": 128, "softcap": 0.0},
        # Softcapped scores, ungrouped heads of 64, odd lengths, FP16.
        {"name": "prefix_decode_softcap", "op": "shared_prefix", "dtype": "f16", "batch": 33, "tokens": 1,
         "prefix": 8191, "suffix": 333, "hq": 16, "hkv": 16, "hd": 64, "softcap": 30.0},
        # Sixteen questions of a hundred tokens read behind a shared document.
        {"name": "prefix_extend", "op": "shared_prefix", "dtype": "bf16", "batch": 16, "tokens": 100, "prefix": 8192,
         "suffix": 512, "hq": 32, "hkv": 8, "hd": 128, "softcap": 0.0},
        # Two sequences behind a very long prefix: few rows, one long axis.
        {"name": "prefix_long", "op": "shared_prefix", "dtype": "bf16", "batch": 2, "tokens": 1, "prefix": 131072,
         "suffix": 1000, "hq": 32, "hkv": 8, "hd": 64, "softcap": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "rope_axes", "shared_prefix"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "shared_prefix":
        hkv, group, hd = rng.choice([2, 4, 8, 16]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        hq = min(32, hkv * group) // hkv * hkv
        prefix = _log(rng, 64, 131072)
        # at most the rows times keys, and the keys, of the largest listed cases
        rows = max(1, min(1600, 16 * 100 * 8192 * 32 * 128 // (prefix * hq * hd)))
        tokens = 1 if rng.random() < 0.6 else _log(rng, 2, max(2, min(128, rows)))
        batch = _log(rng, 1, max(1, min(64, rows // tokens)))
        suffix = tokens + _log(rng, 1, 2047)
        return {"op": op, "dtype": dtype, "batch": batch, "tokens": tokens, "prefix": prefix, "suffix": suffix,
                "hq": hq, "hkv": hkv, "hd": hd, "softcap": rng.choice([0.0, 0.0, 30.0, 50.0])}
    hd = rng.choice([64, 80, 96, 128, 256])
    hq, group = rng.choice([8, 16, 32]), rng.choice([1, 2, 4, 8])
    train = rng.random() < 0.5
    seq = 1 if rng.random() < 0.25 and not train else _log(rng, 2, 8192)
    most = 4 * 4096 * 40 * 128 // ((hq + hq // group) * hd)
    case = {"op": op, "dtype": dtype, "batch": _log(rng, 1, max(1, min(256, most // seq))), "seq": seq, "hq": hq,
            "hkv": hq // group, "hd": hd, "rotary": rng.choice([hd, hd, hd // 2]),
            "interleaved": rng.random() < 0.5, "packed": rng.random() < 0.5, "train": train}
    if op == "qk_norm_rope":
        return {**case, "weight": rng.choice(["same", "f32", "none"])}
    return {**case, "axes": rng.choice([2, 3]), "cyclic": rng.random() < 0.5}


def _dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.bfloat16


def _increments(case):
    """Q0.32 turns per position of the rotary frequencies, as unsigned values."""
    freq = THETA ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
    return torch.round(freq * (TURN / (2 * math.pi))).to(torch.int64)


def _frequency_axes(case):
    """The axis of each frequency: in turn, or in sections, the first half as long."""
    n, axes = case["rotary"] // 2, case["axes"]
    if case["cyclic"]:
        return torch.arange(n) % axes
    first = n // axes if axes == 2 else n // 4
    rest = torch.arange(n - first) * (axes - 1) // (n - first) + 1
    return torch.cat([torch.zeros(first, dtype=torch.int64), rest])


def _video_positions(case, seed):
    """[axes, batch, seq]: text at equal positions on every axis, then a grid."""
    b, s, axes = case["batch"], case["seq"], case["axes"]
    g = torch.Generator().manual_seed(seed)
    start = torch.randint(0, 100000 if s == 1 else 4096, (b, 1), generator=g)
    if s == 1:
        return start.expand(axes, b, 1).clone()
    text = torch.randint(0, max(1, s // 4), (b, 1), generator=g) if axes == 3 else torch.zeros(b, 1, dtype=torch.int64)
    width = max(1, int(round(math.sqrt(s)) * 2 // 3))
    i = torch.arange(s).expand(b, s)
    cell = (i - text).clamp_min(0)
    frame, y, x = cell // (width * width), cell // width % width, cell % width
    grid = torch.stack([frame, y, x]) if axes == 3 else torch.stack([cell // width, x])
    return torch.where(i < text, i, text + grid) + (start if axes == 3 else 0)


def _suffix_lens(case):
    """Valid suffix keys of each sequence, from the new tokens alone to the cache's end."""
    b, t, length = case["batch"], case["tokens"], case["suffix"]
    return [t + (length - t) * i // max(1, b - 1) for i in range(b)] if b > 1 else [length]


def _inputs(case, seed):
    """The operands, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _dtype(case)

    def normal(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)

    b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["hd"]
    if case["op"] == "shared_prefix":
        lens = torch.tensor(_suffix_lens(case), dtype=torch.int32)
        order = torch.randperm(b, generator=torch.Generator().manual_seed(seed))
        # scores that reach a softcap's bend
        return {"q": normal(b, case["tokens"], hq, d, scale=8.0 if case["softcap"] else 1.0),
                "prefix_k": normal(case["prefix"], hkv, d), "prefix_v": normal(case["prefix"], hkv, d),
                "suffix_k": normal(b, case["suffix"], hkv, d), "suffix_v": normal(b, case["suffix"], hkv, d),
                "lens": lens[order].cuda()}
    s = case["seq"]
    if case["packed"]:  # views of the packed projection
        qkv = normal(b, s, (hq + 2 * hkv) * d)
        q = qkv[..., : hq * d].unflatten(-1, (hq, d))
        k = qkv[..., hq * d: (hq + hkv) * d].unflatten(-1, (hkv, d))
    else:
        q, k = normal(b, s, hq, d), normal(b, s, hkv, d)
    x = {"q": q, "k": k, "q_weight": None, "k_weight": None, "axes": None}
    if case["op"] == "rope_axes":
        x["positions"], x["axes"] = _video_positions(case, seed).cuda(), _frequency_axes(case).to(torch.int32).cuda()
    else:
        far = torch.randint(0, 131072 - s, (b, 1), generator=torch.Generator().manual_seed(seed)).cuda()
        x["positions"] = far + torch.arange(s, device="cuda")
        if case["weight"] != "none":
            wt = torch.float32 if case["weight"] == "f32" else dt
            x["q_weight"], x["k_weight"] = (normal(d, scale=0.1, dtype=wt) + 1 for _ in range(2))
    if case["train"]:
        x["dq_out"], x["dk_out"] = normal(b, hq, s, d), normal(b, hkv, s, d)
    return x


def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    if case["op"] != "shared_prefix":
        inc = _increments(case)
        # the storage of a 32-bit phase is signed
        state["inc"] = torch.where(inc >= TURN // 2, inc - TURN, inc).to(torch.int32).cuda()
    if case.get("train"):
        state["leaves"] = [n for n in ("q", "k", "q_weight", "k_weight") if state[n] is not None]
        for n in state["leaves"]:
            state[n] = state[n].detach().requires_grad_(True)
    return state


# ---- the framework's calls ----------------------------------------------------

def _framework():
    path = os.path.join(os.getcwd(), "fast-polynomial-transcendentals_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sfu_repro import fa4_runtime, rope
    return fa4_runtime, rope


def _call(state):
    case = state["case"]
    fa4_runtime, rope = _framework()
    if case["op"] == "shared_prefix":
        return fa4_runtime.flash_attn_shared_prefix(state["q"], state["prefix_k"], state["prefix_v"],
                                                    state["suffix_k"], state["suffix_v"], state["lens"],
                                                    softcap=case["softcap"])
    if case["op"] == "rope_axes":
        return rope.rope_axes(state["q"], state["k"], state["inc"], state["positions"], state["axes"],
                              interleaved=case["interleaved"])
    return rope.qk_norm_rope(state["q"], state["k"], state["q_weight"], state["k_weight"], state["inc"],
                             state["positions"], eps=EPS, interleaved=case["interleaved"])


# ---- the same in elementary operations, in 32 bits ------------------------------

def _cos_sin(state):
    """[batch, seq, 1, frequencies] each; the angles in 64 bits."""
    pos = state["positions"].long()
    if state["axes"] is not None:
        pos = pos.index_select(0, state["axes"].long()).movedim(0, -1)  # the axis of each frequency
    else:
        pos = pos[..., None]
    turns = (pos * (state["inc"].long() % TURN)) % TURN
    angle = turns.double() * (2 * math.pi / TURN)
    return angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)


def _rotate(x, cos, sin, interleaved):
    """The leading 2 * frequencies elements of each head, turned by the angles."""
    n = 2 * cos.shape[-1]
    head, rest = x[..., :n], x[..., n:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., : n // 2], head[..., n // 2:])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    head = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((head, rest), -1)


def _rstd(x):
    return torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_forward(state, x, w, cos, sin):
    y = x.float()
    if state["case"]["op"] == "qk_norm_rope":
        y = y * _rstd(y)
        if w is not None:
            y = y * w.float()
    return _rotate(y, cos, sin, state["case"]["interleaved"]).transpose(1, 2).contiguous().to(x.dtype)


def _plain_backward(state, x, w, dy, cos, sin):
    """(dx, dw), with r the reciprocal root mean square, n = x r and g the
    gradient at n w: dx = r (w g - n mean(w g n)), dw = sum g n."""
    g = _rotate(dy.transpose(1, 2).float(), cos, -sin, state["case"]["interleaved"])
    if state["case"]["op"] == "rope_axes":
        return g.to(x.dtype), None
    f = x.float()
    r = _rstd(f)
    n = f * r
    dw = None if w is None else (g * n).sum((0, 1, 2)).to(w.dtype)
    if w is not None:
        g = g * w.float()
    return (r * (g - n * (g * n).mean(-1, keepdim=True))).to(x.dtype), dw


def _plain_rope(state):
    cos, sin = _cos_sin(state)
    out = [_plain_forward(state, state[n], state[n + "_weight"], cos, sin) for n in ("q", "k")]
    if not state["case"]["train"]:
        return out
    dq, dwq = _plain_backward(state, state["q"], state["q_weight"], state["dq_out"], cos, sin)
    dk, dwk = _plain_backward(state, state["k"], state["k_weight"], state["dk_out"], cos, sin)
    return [*out, dq, dk] + ([] if dwq is None else [dwq, dwk])


def _plain_shared_prefix(state):
    """Token t of sequence b sees the prefix and suffix keys 0 .. lens[b] - T + t."""
    case = state["case"]
    b, t, hq, hkv, d = case["batch"], case["tokens"], case["hq"], case["hkv"], case["hd"]
    p, length, group = case["prefix"], case["suffix"], hq // hkv
    q = state["q"].float().mul(1 / math.sqrt(d)).view(b, t, hkv, group, d).permute(2, 0, 1, 3, 4).contiguous()
    pk, pv = (state[n].float().transpose(0, 1).contiguous() for n in ("prefix_k", "prefix_v"))        # [hkv, p, d]
    sk, sv = (state[n].float().transpose(1, 2).contiguous().transpose(0, 1).contiguous()
              for n in ("suffix_k", "suffix_v"))                                                      # [hkv, b, l, d]
    sp = torch.matmul(q.view(hkv, -1, d), pk.transpose(1, 2).contiguous()).view(hkv, b, t * group, p)
    ss = torch.matmul(q.view(hkv, b, t * group, d), sk.transpose(2, 3).contiguous())                  # [.., l]
    if case["softcap"]:
        sp, ss = (torch.tanh(x / case["softcap"]) * case["softcap"] for x in (sp, ss))
    seen = state["lens"].long()[:, None] - t + 1 + torch.arange(t, device="cuda")                     # [b, t]
    hidden = torch.arange(length, device="cuda") >= seen[..., None]                                   # [b, t, l]
    hidden = hidden[:, :, None].expand(b, t, group, length).reshape(b, t * group, length)
    ss = ss.masked_fill(hidden, -math.inf)
    m = torch.maximum(sp.amax(-1, keepdim=True), ss.amax(-1, keepdim=True))
    ep, es = torch.exp(sp - m), torch.exp(ss - m)
    total = ep.sum(-1, keepdim=True) + es.sum(-1, keepdim=True)
    out = torch.matmul(ep.view(hkv, -1, p), pv).view(hkv, b, t * group, d) + torch.matmul(es, sv)
    out = (out / total).view(hkv, b, t, group, d).permute(1, 2, 0, 3, 4).reshape(b, t, hq, d)
    lse = (m + torch.log(total)).view(hkv, b, t, group).permute(1, 0, 3, 2).reshape(b, hq, t)
    return [out.to(state["q"].dtype), lse]


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _plain_shared_prefix(state) if case["op"] == "shared_prefix" else _plain_rope(state)
    if not case.get("train"):
        with torch.no_grad():
            return list(_call(state))
    out = _call(state)
    grads = torch.autograd.grad(out, [state[n] for n in state["leaves"]], [state["dq_out"], state["dk_out"]])
    return [*(o.detach() for o in out), *grads]


def work(case):
    b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["hd"]
    if case["op"] == "shared_prefix":
        t, lens = case["tokens"], _suffix_lens(case)
        rows, keys = b * t * hq, case["prefix"] + sum(lens)
        pairs = b * t * case["prefix"] + sum(t * n - t * (t - 1) // 2 for n in lens)
        # Q, O, the prefix once, each sequence's own keys; two products
        return {"bytes": 4 * rows * d + 4 * rows + 4 * keys * hkv * d + 4 * b, "flops": 4 * hq * d * pairs}
    n, tokens = b * case["seq"] * (hq + hkv) * d, b * case["seq"]
    norm = case["op"] == "qk_norm_rope"
    # x -> y; with training dy -> dx, and x again where a norm's gradient needs it
    streams = 2 + (0 if not case["train"] else 3 if norm else 2)
    return {"bytes": 2 * n * streams + 8 * tokens * case.get("axes", 1),
            "flops": n * (7 if norm else 3) * (3 if case["train"] and norm else 2 if case["train"] else 1)}


# ---- the definitions in 64 bits ---------------------------------------------------

def _exact_rope(case, x):
    inc = _increments(case).cuda()
    pos = x["positions"].long()
    if x["axes"] is not None:
        pos = torch.stack([pos[a] for a in x["axes"].tolist()], -1)
    else:
        pos = pos.unsqueeze(-1)
    angle = torch.remainder(pos * inc, TURN).double() * (2 * math.pi / TURN)
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(2)  # e^{i angle}
    r = case["rotary"]
    leaves = {n: x[n].double().requires_grad_(case["train"]) for n in ("q", "k", "q_weight", "k_weight")
              if x[n] is not None}
    outs = []
    with torch.set_grad_enabled(case["train"]):
        for n in ("q", "k"):
            y = leaves[n]
            if case["op"] == "qk_norm_rope":
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["hd"] + EPS) * leaves.get(n + "_weight", 1.0)
            pairs = y[..., :r].unflatten(-1, (-1, 2)) if case["interleaved"] else y[..., :r].unflatten(-1, (2, -1)).mT
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            z = (z if case["interleaved"] else z.mT).flatten(-2)
            outs.append(torch.cat((z, y[..., r:]), -1).transpose(1, 2))
    if not case["train"]:
        return outs
    grads = torch.autograd.grad(outs, list(leaves.values()), [x["dq_out"].double(), x["dk_out"].double()])
    return [*(o.detach() for o in outs), *grads]


def _exact_shared_prefix(case, x):
    b, t, hq, d, group = case["batch"], case["tokens"], case["hq"], case["hd"], case["hq"] // case["hkv"]
    out = torch.empty(b, t, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.empty(b, hq, t, dtype=torch.float64, device="cuda")
    lens = x["lens"].tolist()
    rows = max(1, (1 << 27) // ((case["prefix"] + case["suffix"]) * group * t))  # sequences at a time
    for h in range(case["hkv"]):
        heads = slice(h * group, (h + 1) * group)
        pk, pv = x["prefix_k"][:, h].double(), x["prefix_v"][:, h].double()
        for b0 in range(0, b, rows):
            q = x["q"][b0:b0 + rows, :, heads].double()                      # [n, t, g, d]
            n = q.shape[0]
            far = (q.reshape(-1, d) @ pk.t().contiguous()).view(n, t, group, -1)
            near = torch.full((n, t, group, case["suffix"]), -math.inf, dtype=torch.float64, device="cuda")
            for i in range(n):
                c = lens[b0 + i]
                s = q[i].reshape(-1, d) @ x["suffix_k"][b0 + i, :c, h].double().t().contiguous()
                cut = torch.ones(t, c, dtype=torch.bool, device="cuda").triu(c - t + 1)
                near[i, :, :, :c] = s.view(t, group, c).masked_fill(cut[:, None], math.nan)
            s = torch.cat((far, near), -1) / math.sqrt(d)
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
                s[..., case["prefix"]:].masked_fill_(near == -math.inf, -math.inf)
            s = s.nan_to_num_(nan=-math.inf, neginf=-math.inf)
            z = torch.logsumexp(s, -1)
            s.sub_(z[..., None]).exp_()
            o = (s[..., : case["prefix"]].reshape(-1, case["prefix"]) @ pv).view(n, t, group, d)
            for i in range(n):
                c = lens[b0 + i]
                own_v = x["suffix_v"][b0 + i, :c, h].double()
                o[i] += (s[i, :, :, case["prefix"]: case["prefix"] + c].reshape(-1, c) @ own_v).view(t, group, d)
            out[b0:b0 + n, :, heads] = o
            lse[b0:b0 + n, heads] = z.transpose(1, 2)
    return [out, lse]


def exact(case, seed):
    """The operators' definitions, in 64 bits."""
    x = _inputs(case, seed)
    return _exact_shared_prefix(case, x) if case["op"] == "shared_prefix" else _exact_rope(case, x)
