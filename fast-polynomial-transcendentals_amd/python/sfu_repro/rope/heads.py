"""Query and key heads between their projection and the attention: the norm of
each head, the rotary rotation by positions that the caller gives, on one axis
or several, and their gradients.

The reference rotates interleaved pairs by the positions 0..S-1 and leaves the
norm to the model (``src/sfu_repro/rope/benchmark_cuda_fused_rope.py:71-97``,
``src/sfu_repro/fa4.py:500-549``); these operators have no counterpart there.
They keep the layout of ``spline_ops.rope_apply_*``: q ``[batch, sequence,
heads, head_dim]`` in, ``[batch, heads, sequence, head_dim]`` out, phase
increments in Q0.32 turns per position.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch


@lru_cache(maxsize=1)
def _ops():
    """The compiled extension; fails loudly when it is missing."""
    try:
        import spline_ops
    except (ImportError, OSError) as error:
        raise RuntimeError(
            "The compiled spline_ops extension (libspline_hip.so) is unavailable. Build it with "
            "`python fast-polynomial-transcendentals_amd/build.py`.") from error
    return spline_ops


def phase_increments(rotary_dim: int, theta: float = 10000.0, *, device=None) -> torch.Tensor:
    """int32 ``[rotary_dim / 2]``: the frequencies ``theta ** (-2i / rotary_dim)``
    in units of 2^-32 turns per position."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    freq = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(rotary_dim, 1))
    turns = torch.round(freq * (2.0 ** 32 / (2 * math.pi))).to(torch.int64) % 2 ** 32
    return torch.where(turns >= 2 ** 31, turns - 2 ** 32, turns).to(torch.int32).to(device)


def axis_sections(sections, *, device=None) -> torch.Tensor:
    """``frequency_axes`` whose first ``sections[0]`` frequencies turn by axis 0,
    the next ``sections[1]`` by axis 1, and so on."""
    counts = [int(n) for n in sections]
    if not counts or min(counts) < 0:
        raise ValueError(f"sections must be the frequencies of each axis, got {sections!r}")
    return torch.cat([torch.full((n,), axis, dtype=torch.int32) for axis, n in enumerate(counts)]).to(device)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 phase_increments: torch.Tensor, positions: torch.Tensor | None = None, *,
                 frequency_axes: torch.Tensor | None = None, eps: float = 1e-6,
                 interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head, times its weight, then the rotary
    rotation, in one pass; differentiable in q, k and the weights.

    ``q [B, S, Hq, D]`` and ``k [B, S, Hk, D]``, float16 or bfloat16, any strides
    (views of a packed projection take no copy), D a multiple of 8 up to 256;
    returns ``[B, Hq, S, D]`` and ``[B, Hk, S, D]``.  The weights ``[D]`` are
    float32 or of q's type, ``None`` for ones.  ``phase_increments`` int32
    ``[R / 2]`` turns the first R elements of a head (R a multiple of 8, at most
    D); the pairs are ``(2i, 2i + 1)``, or ``(i, i + R / 2)`` with
    ``interleaved=False``.  ``positions`` int32 or int64, any values: ``[S]`` or
    ``[B, S]``, ``None`` for 0..S-1, or ``[axes, B, S]`` with ``frequency_axes``
    (see :func:`rope_axes`).
    """
    return tuple(_ops().qk_norm_rope_ag(q, k, q_weight, k_weight, phase_increments, positions, frequency_axes,
                                        float(eps), bool(interleaved)))


def rope_axes(q: torch.Tensor, k: torch.Tensor, phase_increments: torch.Tensor, positions: torch.Tensor,
              frequency_axes: torch.Tensor, *, interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """The rotary rotation by positions of several axes (time, height, width);
    differentiable in q and k.

    ``positions [axes, B, S]``; frequency i turns by the position on axis
    ``frequency_axes[i]`` (int32 ``[R / 2]``, held to the axes that there are;
    :func:`axis_sections` builds one of consecutive sections).  Operands, pairs
    and layouts are those of :func:`qk_norm_rope`.
    """
    return tuple(_ops().rope_axes_ag(q, k, phase_increments, positions, frequency_axes, bool(interleaved)))


__all__ = ["axis_sections", "phase_increments", "qk_norm_rope", "rope_axes"]
