"""Paired sine/cosine evaluation for rotary embeddings on the MI355X
(counterpart of the reference's src/sfu_repro/rope/).

Importing this package performs no model or runtime monkey-patching.
"""

from .heads import axis_sections, phase_increments, qk_norm_rope, rope_axes

__all__ = ["axis_sections", "phase_increments", "qk_norm_rope", "rope_axes"]
