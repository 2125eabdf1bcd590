"""Host side of the cache in pages of 4-bit numbers: what its entry points refuse before they
launch anything, their workspaces, and the definitions that the GPU tests compare with (runs
without a GPU)."""

import ctypes
import math

import pytest
import torch

import capi_helpers
import paged_reference as ref


class Cache(ctypes.Structure):
    """spline_hip_fp4_cache."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("cache", "table", "lens")]
                + [(n, ctypes.c_int64) for n in ("pages", "page_size", "kv_heads", "head_dim", "batch", "entries",
                                                 "table_stride")])


class Attention(ctypes.Structure):
    """spline_hip_fp4_attention."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("out", "lse", "q", "workspace")]
                + [(n, ctypes.c_int64) for n in ("tokens", "q_heads")] + [("q_strides", ctypes.c_int64 * 3)]
                + [("mode", ctypes.c_int32), ("scale", ctypes.c_float), ("cap", ctypes.c_float)])


class Pages(ctypes.Structure):
    """spline_hip_pages."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("out_table", "out_lens", "out_count", "table", "lens", "parents", "caches",
                                                "cache_page_bytes", "workspace")]
                + [(n, ctypes.c_int64) for n in ("num_caches", "old_rows", "rows", "entries", "table_stride", "pages",
                                                 "page_size", "grow")])


def _cache(**changes):
    c = Cache(cache=4096, table=4096, lens=4096, pages=100, page_size=64, kv_heads=2, head_dim=128, batch=3, entries=10,
              table_stride=10)
    for name, value in changes.items():
        setattr(c, name, value)
    return ctypes.byref(c)


def _attention(**changes):
    a = Attention(out=4096, lse=4096, q=4096, workspace=4096, tokens=1, q_heads=8, mode=0, scale=0.1, cap=30.0)
    for name, value in changes.items():
        setattr(a, name, value)
    return ctypes.byref(a)


PTRS = (ctypes.c_void_p * 2)(4096, 8192)
BYTES = (ctypes.c_int64 * 2)(64, 160)


def _pages(ptrs=PTRS, sizes=BYTES, **changes):
    a = Pages(out_table=4096, out_lens=4096, out_count=4096, table=4096, lens=4096, parents=4096,
              caches=ctypes.cast(ptrs, ctypes.c_void_p), cache_page_bytes=ctypes.cast(sizes, ctypes.c_void_p),
              workspace=4096, num_caches=2, old_rows=4, rows=4, entries=5, table_stride=5, pages=100, page_size=64, grow=1)
    for name, value in changes.items():
        setattr(a, name, value)
    return ctypes.byref(a)


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(capi_helpers.LIB)
    for name in ("spline_hip_paged_fp4_workspace_bytes", "spline_hip_fork_pages_workspace_bytes",
                 "spline_hip_compact_pages_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_int64
    return lib


def _id(c):
    return "-".join(f"{k}-{v}" for k, v in c.items() if isinstance(v, (int, float, type(None))))


SIZES = [dict(pages=-1), dict(pages=2 ** 31), dict(page_size=0), dict(page_size=24), dict(page_size=-16),
         dict(page_size=65552), dict(kv_heads=0), dict(kv_heads=2 ** 17), dict(head_dim=96), dict(batch=-1),
         dict(batch=2 ** 31), dict(entries=-1), dict(entries=2 ** 24 + 1), dict(entries=2 ** 60)]
POINTERS = [dict(cache=None), dict(cache=4104), dict(table=None), dict(table=4098), dict(lens=None), dict(lens=4098),
            dict(table_stride=-1)]


@pytest.mark.parametrize("bad", SIZES + POINTERS, ids=_id)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_caches_are_refused(lib, bad, dtype):
    s = (ctypes.c_int64 * 3)(256, 256, 128)
    p = ctypes.c_void_p(4096)
    t = ctypes.c_int64(1)
    assert getattr(lib, f"launch_paged_fp4_store_{dtype}")(_cache(**bad), p, p, s, s, t, None) == 1
    assert getattr(lib, f"launch_paged_fp4_load_{dtype}")(_cache(**bad), p, p, t, None) == 1
    assert getattr(lib, f"launch_paged_fp4_attention_{dtype}")(_cache(**bad), _attention(), None) == 1


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_are_refused(lib, dtype):
    store, load = (getattr(lib, f"launch_paged_fp4_{n}_{dtype}") for n in ("store", "load"))
    s = (ctypes.c_int64 * 3)(256, 256, 128)
    good, one = ctypes.c_void_p(4096), ctypes.c_int64(1)
    for k, v in ((None, good), (good, None), (ctypes.c_void_p(4104), good), (good, ctypes.c_void_p(4100))):
        assert store(_cache(), k, v, s, s, one, None) == 1
        assert load(_cache(), k, v, one, None) == 1
    for odd in ((ctypes.c_int64 * 3)(256, 4, 128), (ctypes.c_int64 * 3)(-256, 256, 128), None):
        assert store(_cache(), good, good, odd, s, one, None) == 1
        assert store(_cache(), good, good, s, odd, one, None) == 1
    for tokens in (-1, 2 ** 14 + 1):
        assert store(_cache(), good, good, s, s, ctypes.c_int64(tokens), None) == 1
        assert load(_cache(), good, good, ctypes.c_int64(tokens), None) == 1
    assert store(_cache(batch=2 ** 24, kv_heads=16), good, good, s, s, ctypes.c_int64(4), None) == 1  # more than 2^32 threads
    for nothing in (dict(batch=0), dict()):
        t = ctypes.c_int64(1 if nothing else 0)
        assert store(_cache(**nothing), good, good, s, s, t, None) == 0
        assert load(_cache(**nothing), good, good, t, None) == 0
    assert store(None, good, good, s, s, one, None) == 1 and load(None, good, good, one, None) == 1


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(tokens=2 ** 14 + 1), dict(q_heads=0), dict(q_heads=7), dict(q_heads=2 ** 17), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(mode=1), dict(mode=5), dict(mode=-1),
    dict(mode=3, cap=0.0), dict(mode=3, cap=float("inf")), dict(q=None), dict(q=4104), dict(out=None), dict(out=4104),
    dict(lse=4098), dict(workspace=None), dict(workspace=4104), dict(q_strides=(ctypes.c_int64 * 3)(8, 8, 4)),
    dict(q_strides=(ctypes.c_int64 * 3)(-8, 8, 8))], ids=_id)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attentions_are_refused(lib, bad, dtype):
    assert getattr(lib, f"launch_paged_fp4_attention_{dtype}")(_cache(), _attention(**bad), None) == 1


def test_attention_of_nothing(lib):
    for dtype in ("fp16", "bf16"):
        call = getattr(lib, f"launch_paged_fp4_attention_{dtype}")
        assert call(_cache(batch=0), _attention(), None) == 0 and call(_cache(), _attention(tokens=0), None) == 0
        assert call(None, _attention(), None) == 1 and call(_cache(), None, None) == 1
    assert lib.launch_paged_fp4_attention_fp16(_cache(), _attention(mode=4), None) == 1  # a BF16 program


def test_attention_workspace(lib):
    """It goes by the rows of a tile and the device, not by keys or sequences."""
    size = lambda c=None, **a: lib.spline_hip_paged_fp4_workspace_bytes(_cache(**(c or {})), _attention(**a))  # noqa: E731
    assert size() > 0 and size() % 16 == 0
    assert size(dict(entries=2 ** 24)) == size(dict(batch=1000)) == size()
    assert size(dict(batch=0)) == size(tokens=0) == 0
    for bad in SIZES:
        assert size(bad) == -1, bad
    assert size(tokens=-1) == size(q_heads=7) == size(dict(batch=2 ** 30), tokens=2 ** 14) == -1


PAGE_SIZES = [dict(rows=-1), dict(old_rows=-1), dict(rows=2 ** 24 + 1), dict(entries=-1), dict(entries=2 ** 24 + 1),
              dict(pages=-1), dict(pages=2 ** 31), dict(num_caches=-1), dict(rows=2 ** 20, old_rows=2 ** 20, entries=2 ** 14)]
FORK_SIZES = [dict(page_size=0), dict(page_size=-1), dict(page_size=2 ** 17), dict(grow=-1), dict(grow=2 ** 30)]


@pytest.mark.parametrize("bad", PAGE_SIZES + [
    dict(out_table=None), dict(out_table=4098), dict(out_count=None), dict(table=None), dict(table=4098),
    dict(table_stride=-1), dict(workspace=None), dict(workspace=4104), dict(caches=None), dict(cache_page_bytes=None),
    dict(ptrs=(ctypes.c_void_p * 2)(4096, None)), dict(ptrs=(ctypes.c_void_p * 2)(4104, 4096)),
    dict(sizes=(ctypes.c_int64 * 2)(64, 40)), dict(sizes=(ctypes.c_int64 * 2)(-16, 64)),
    dict(sizes=(ctypes.c_int64 * 2)(16, 2 ** 50))], ids=_id)
def test_pages_are_refused(lib, bad):
    assert lib.launch_fork_pages(_pages(**bad), None) == 1
    assert lib.launch_compact_pages(_pages(**bad), None) == 1


@pytest.mark.parametrize("bad", FORK_SIZES + [dict(out_lens=None), dict(out_lens=4098), dict(lens=None), dict(lens=4098),
                                              dict(parents=4098), dict(parents=None, rows=3)], ids=_id)
def test_forks_are_refused(lib, bad):
    assert lib.launch_fork_pages(_pages(**bad), None) == 1


def test_page_workspaces(lib):
    fork, compact = lib.spline_hip_fork_pages_workspace_bytes, lib.spline_hip_compact_pages_workspace_bytes
    assert fork(_pages()) > 0 and compact(_pages()) > 0
    for bad in PAGE_SIZES:
        assert fork(_pages(**bad)) == -1 and compact(_pages(**bad)) == -1, bad
    for bad in FORK_SIZES:
        assert fork(_pages(**bad)) == -1, bad
    assert compact(_pages(rows=3)) == -1  # compacting keeps the rows
    assert fork(None) == -1 and compact(None) == -1
    assert lib.launch_fork_pages(None, None) == 1 and lib.launch_compact_pages(None, None) == 1


def test_wishes_are_counted_in_32_bits(lib):
    size = lib.spline_hip_fork_pages_workspace_bytes
    rows = dict(rows=2 ** 20, old_rows=2 ** 20, entries=6, page_size=64)
    assert size(_pages(**rows, grow=64 * 2000)) > 0  # 2^20 rows of 6 + 2 + 2000 pages
    for grow in (64 * 2040, 2 ** 28):
        assert size(_pages(**rows, grow=grow)) == -1
        assert lib.launch_fork_pages(_pages(**rows, grow=grow), None) == 1


def test_python_refuses_host_tensors():
    from sfu_repro import fa4_runtime, paged_cache

    cache = paged_cache.fp4_cache(3, 2, 64, 16)
    assert cache.shape == (3, 2, 2, 16 * 34)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: fa4_runtime.flash_attn_paged_fp4(q, cache, table, lens),
                 lambda: paged_cache.store_fp4(cache, q, q, table, lens),
                 lambda: paged_cache.load_fp4(cache, table, lens, 1, 64),
                 lambda: paged_cache.fork_pages([cache], table, lens, page_size=16),
                 lambda: paged_cache.compact_pages([cache], table)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_caches_of_other_shapes_are_refused():
    from sfu_repro import paged_cache

    for args in ((3, 2, 96), (3, 2, 64, 24), (3, 2, 64, 0), (3, 2, 128, 2 ** 17)):
        with pytest.raises(ValueError):
            paged_cache.fp4_cache(*args)


def test_gradients_are_refused():
    from torch.autograd import forward_ad
    from sfu_repro import fa4_runtime, paged_cache

    cache = paged_cache.fp4_cache(3, 2, 64, 16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    calls = (lambda x: fa4_runtime.flash_attn_paged_fp4(x, cache, table, lens),
             lambda x: paged_cache.store_fp4(cache, x, q, table, lens), lambda x: paged_cache.store_fp4(cache, q, x, table, lens))
    for call in calls:
        with pytest.raises(RuntimeError, match="has no backward"):
            call(q.clone().requires_grad_(True))
        with torch.no_grad(), forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
                call(forward_ad.make_dual(q, torch.ones_like(q)))


# ---- the definitions ------------------------------------------------------------------


def test_numbers_of_a_cache():
    cache = torch.zeros(1, 2, 1, 16 * 34, dtype=torch.uint8)
    cache[0, 0, 0, 16 * 32:] = 127
    cache[0, 0, 0, 32] = 0xA7            # row 1, elements 0 and 1: 6 and -1
    cache[0, 0, 0, 32 + 16] = 0x0D       # element 32: -3
    cache[0, 0, 0, 16 * 32 + 2: 16 * 32 + 4] = torch.tensor([128, 125], dtype=torch.uint8)
    v = ref.numbers(cache, 64)
    assert v[0, 0, 0, 1, :2].tolist() == [12, -2] and v[0, 0, 0, 1, 32] == -0.75
    assert float(v[0, 0].abs().sum()) == 14.75
    cache[0, 1, 0, -1] = 253
    assert bool(ref.numbers(cache, 64)[0, 1, 0, 15, 32:].isnan().all()) and int(ref.numbers(cache, 64).isnan().sum()) == 32


def test_nearest_numbers():
    x = torch.zeros(32)
    x[:9] = torch.tensor([6.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.26])
    assert ref.nearest(x)[:9].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -0.5]
    x[0] = 7.0  # the next power: 3.5 of it
    assert ref.nearest(x)[:4].tolist() == [8, 0, 1, 1]
    assert ref.nearest(torch.full((32,), 3.0e38))[0] == 6 * 2.0 ** 125
    assert ref.nearest(torch.full((32,), 2.0 ** -101))[0] == 2.0 ** -101 and ref.nearest(torch.full((32,), 2.0 ** -102))[0] == 0
    x[5] = math.inf
    assert bool(ref.nearest(x).isnan().all())


def test_forking_and_compacting():
    table = torch.tensor([[4, 7, -1], [2, -1, -1]], dtype=torch.int32)
    lens = torch.tensor([20, 16], dtype=torch.int32)
    new = torch.tensor([0, 0, 1, -1], dtype=torch.int32)
    out, n, short, moves = ref.fork(table, lens, new, 1, 16, 9)
    assert out.tolist() == [[4, 7, -1], [4, 0, -1], [2, 1, -1], [-1, -1, -1]]
    assert n.tolist() == [20, 20, 16, 0] and short == 0 and moves == [(7, 0)]
    assert ref.compact(out, 9)[0].tolist() == [[4, 3, -1], [4, 0, -1], [2, 1, -1], [-1, -1, -1]]
    assert ref.compact(out, 9)[1:] == (5, [(7, 3)])


def test_one_tensor_is_not_a_list_of_caches():
    from sfu_repro import paged_cache

    cache, table, lens = paged_cache.fp4_cache(2, 2, 64, 16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="sequence of caches"):
        paged_cache.fork_pages(cache, table, lens, page_size=16)
    with pytest.raises(TypeError, match="sequence of caches"):
        paged_cache.compact_pages(cache, table)
