"""How the attention over 4-bit pages cuts the keys of its calls: each unit's pieces, as the workspace of a
call through the C entry point tells them."""

import ctypes
import math

import pytest
import torch

import capi_helpers
import paged_reference as ref
from test_gpu_paged_large import _make
from test_paged_cache_cpu import Attention, Cache

pytestmark = pytest.mark.gpu

# dtype, tokens, hq, hkv, dim, page_size, cap, lens; keys of a step
CASES = [
    (("bf16", 1, 8, 1, 64, 64, 0.0, [131072] + [100] * 15), 256),
    (("bf16", 1, 8, 1, 128, 64, 0.0, [100] * 15 + [131072]), 128),
    (("f16", 1, 8, 2, 64, 32, 30.0, [20000] + [50] * 63), 256),
    (("bf16", 40, 8, 2, 128, 64, 0.0, [20000, 100, 41, 90, 100, 64, 100, 70]), 64),
    (("bf16", 1, 8, 1, 128, 64, 0.0, [131072]), 128),
    (("bf16", 1, 32, 8, 128, 64, 0.0, [3000 + i for i in range(16)]), 128),
]


@pytest.mark.parametrize("case,step", CASES, ids=lambda c: "-".join(map(str, c[:7])) if isinstance(c, tuple) else str(c))
def test_a_unit_has_no_more_pieces_than_its_join_takes(cuda, case, step):
    """64 pieces, one for every 32 steps and one more, whatever is beside it: one long sequence among short
    ones too.  The result is that of the definition."""
    dtype, tokens, hq, hkv, dim, size, cap, lens = case
    q, cache, table, n = _make(case, cuda)
    lib = ctypes.CDLL(capi_helpers.LIB)
    lib.spline_hip_paged_fp4_workspace_bytes.restype = ctypes.c_int64
    c = Cache(cache=cache.data_ptr(), table=table.data_ptr(), lens=n.data_ptr(), pages=cache.shape[0], page_size=size,
              kv_heads=hkv, head_dim=dim, batch=len(lens), entries=table.shape[1], table_stride=table.stride(0))
    out, lse = torch.empty_like(q), torch.empty(len(lens), hq, tokens, device=cuda)
    a = Attention(out=out.data_ptr(), lse=lse.data_ptr(), q=q.data_ptr(), tokens=tokens, q_heads=hq,
                  q_strides=(ctypes.c_int64 * 3)(*q.stride()[:3]), mode=3 if cap else 0, scale=1 / math.sqrt(dim), cap=cap)
    total = lib.spline_hip_paged_fp4_workspace_bytes(ctypes.byref(c), ctypes.byref(a))
    work = torch.empty(total, dtype=torch.uint8, device=cuda)
    a.workspace = work.data_ptr()
    call = getattr(lib, f"launch_paged_fp4_attention_{'bf16' if dtype == 'bf16' else 'fp16'}")
    assert call(ctypes.byref(c), ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    rows = tokens * hq // hkv
    tile = next(r for r in (16, 32, 64, 128) if rows <= r or r == 128)
    blocks = total // (16 + 2 * tile * (dim + 2) * 4)  # behind the rows of two pieces a block: batch, .., pieces, row
    cuts = work[total - 16 * blocks:].view(torch.int32).view(blocks, 4).tolist()
    assert any(x[2] for x in cuts) and all(0 <= x[2] <= blocks and 0 <= x[0] < len(lens) for x in cuts)
    for b, _, pieces, _ in cuts:
        steps = -(-lens[b] // step) + 4
        assert pieces <= 64 + steps / 32 + 2, (b, pieces)
    ref.check((out, lse), ref.attention_at_scale(q, cache, table, n, 1 / math.sqrt(dim), cap))
