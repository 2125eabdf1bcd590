"""Sizes that the attention over 4-bit pages takes and refuses (runs without a GPU)."""

from test_paged_cache_cpu import _attention, _cache, lib  # noqa: F401


def test_tokens_past_two_to_the_14(lib):  # noqa: F811
    """They have to fit a row of the table, their rows 2^30."""
    size = lambda c=None, **a: lib.spline_hip_paged_fp4_workspace_bytes(_cache(**(c or {})), _attention(**a))  # noqa: E731
    assert size(tokens=2 ** 14) > 0 and size(tokens=2 ** 14 + 1) == -1  # a row holds 640
    assert size(dict(entries=257), tokens=257 * 64) > 0 and size(dict(entries=257), tokens=257 * 64 + 1) == -1
    long = dict(batch=1, entries=2 ** 20, kv_heads=1)
    assert size(dict(long, entries=2 ** 13), tokens=2 ** 17, q_heads=16) > 0  # 2^14 tiles of 2^13 steps
    assert size(long, tokens=2 ** 26, q_heads=32) == -1  # 2^31 rows
    assert size(long, tokens=2 ** 40) == -1 and size(long, tokens=2 ** 62) == -1
