"""A serving cache in pages of 4-bit numbers, and its pages.

A cache (one a layer) is a uint8 tensor ``[pages, 2, kv_heads, bytes]``: keys and
values of ``page_size`` tokens a page and KV head as E2M1 numbers, in blocks of 32
along the head that share a power of two, 4.25 bits an element (the bytes are laid out
in ``spline_ops_hip.h``).  A sequence's keys lie in the pages that its row of
``table`` names (int32 ``[B, entries]``, -1 for none): the one at position x in row
``x % page_size`` of page ``table[b, x // page_size]``.  ``lens`` (int32 ``[B]``)
counts its keys.  Tables and lengths stay on the device, and so does what decides about
pages: no call waits for the GPU, and all can be captured into a graph.

A decoding step, with ``fa4_runtime.flash_attn_paged_fp4``::

    table, lens, short = fork_pages(caches, table, lens, tokens=1, page_size=64)
    lens = lens + 1
    for each layer: store_fp4(cache, k, v, table, lens)
                    out, lse = flash_attn_paged_fp4(q, cache, table, lens)

The reference has no cache of its own; these operators have no counterpart there.
"""

from __future__ import annotations

from functools import lru_cache

import torch

BLOCK = 32  # elements that share a power of two


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


def _several(caches) -> list:
    if isinstance(caches, torch.Tensor):  # a list of its pages
        raise TypeError("caches must be a sequence of caches, one a layer, not one tensor")
    return list(caches)


def fp4_cache(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, *, device=None) -> torch.Tensor:
    """A cache of ``pages`` pages, all zeros.  head_dim 64 or 128, page_size a multiple of 16."""
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    if page_size <= 0 or page_size % 16 or page_size > 65536:
        raise ValueError(f"page_size must be a multiple of 16 up to 65536, got {page_size}")
    return torch.zeros(pages, 2, kv_heads, page_size * (head_dim // 2 + head_dim // BLOCK), dtype=torch.uint8,
                       device=device)


def store_fp4(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor) -> None:
    """Stores the keys and values ``[B, T, Hkv, D]`` (float16 or bfloat16, any strides)
    of the last T tokens of each sequence: token t at position ``lens[b] - T + t``.

    Tokens whose position is negative (left-padded batches), past the table or on an entry
    without a page are left out; more than 16384 of them have to fit a row of the table, and a call
    holds fewer than 2^34 elements of keys.  A block's power of two 2^e puts its largest
    magnitude into [3.5, 7) 2^e (-100 <= e <= 125); values are rounded to nearest, ties to even,
    the largest number being 6 2^e.  A block with an infinity or NaN reads as NaN.  A page that
    is written belongs to one sequence (:func:`fork_pages` sees to it): of two tokens of a call
    at one place either's bytes stay.
    """
    _ops().paged_fp4_store(cache, k, v, table, lens)


def load_fp4(cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, tokens: int, head_dim: int, *,
             dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values ``[B, tokens, Hkv, head_dim]`` that the cache holds of the last
    ``tokens`` tokens of each sequence: exact in bfloat16, rounded and held to 65504 in float16;
    zeros where a token has no place.  As many tokens as :func:`store_fp4` takes.  ``head_dim`` is the
    one that was stored: pages of 64 rows of 128 elements read as pages of 128 rows of 64."""
    return tuple(_ops().paged_fp4_load(cache, table, lens, int(tokens), int(head_dim), dtype))


def fork_pages(caches, table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor | None = None, *,
               tokens: int = 0, page_size: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(table, lens, short)`` of new rows that continue old ones, with room for
    ``tokens`` more keys each.

    New row i continues row ``parents[i]`` (int32, on the device; ``None``: row i) with its ``lens``
    keys, held to the table.  An id outside the rows is a place in the batch that nothing
    uses: it gets no pages, whatever ``tokens`` is, and counts nothing in ``short``.  A new sequence
    continues a row of no keys, which the table keeps for it (``lens`` 0; several may continue the same one).  A row may be
    continued by several, which share the pages that it has filled; the page that
    the next key goes to belongs to one row, the first that continues it, and is copied
    for every other, in each of ``caches`` (tensors of any kind ``[pages, ...]``, one a layer,
    written in place).  A page is in use where a row names it: pages of rows that
    nobody continues, and entries behind a row's keys, are free behind the call, so
    ending a sequence is leaving it out, taking keys back is lowering its ``lens``, and
    rows may hold prefixes that nothing decodes.  New pages are the lowest free ones, in the
    order of rows and entries; other entries are -1.

    ``page_size`` is the keys of a page in every one of ``caches``: a wrong one would share pages that are
    still written.  Caches of :func:`fp4_cache` whose pages have not the bytes for it are refused (pages
    of 64 rows of 128 elements have those of 128 rows of 64); what other caches hold is the caller's
    (one of their shape, uint8 ``[pages, 2, heads, 544 n]``, is passed as ``cache.flatten(1)``).

    ``short`` (int32 ``[1]``) counts the pages that were wanted and not to be had, entries past
    the table's width among them; their entries are -1, and a row whose copy is missing has lost the
    keys of its last page.  The table and lengths given are left as they are.
    """
    return tuple(_ops().fork_pages(_several(caches), table, lens, parents, int(tokens), int(page_size)))


def compact_pages(caches, table: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(table, used)``: moves the pages that ``table`` names to the front of every cache
    (as in :func:`fork_pages`, written in place).  Of ``used`` pages (int32 ``[1]``) those with
    numbers from ``used`` on move to the free ones below, both in ascending order; entries
    that named no page are -1.  The table given is left as it is."""
    return tuple(_ops().compact_pages(_several(caches), table))


__all__ = ["compact_pages", "fork_pages", "fp4_cache", "load_fp4", "store_fp4"]
