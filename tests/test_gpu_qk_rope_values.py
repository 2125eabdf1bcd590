"""Head norm at the ends of what its operands hold: weights that are no numbers,
sides and batches without a row."""

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rotary", [0, 16, 24])
@pytest.mark.parametrize("inter", [True, False])
def test_infinite_weights_behind_the_rotated_elements(cuda, inter, rotary, dtype):
    """What is not turned is x r w: an infinite weight gives an infinity of x's
    sign there, and every other element keeps its bits."""
    from sfu_repro import rope

    g = torch.Generator().manual_seed(30)
    q, k = (torch.randn(2, 9, h, 48, generator=g).to(torch.float16).to(cuda) for h in (3, 2))
    q[q == 0], k[k == 0] = 1, 1
    w = (1 + 0.2 * torch.randn(48, generator=g)).to(dtype).to(cuda)
    inc = rope.phase_increments(rotary, 500000.0).to(cuda)
    clean = rope.qk_norm_rope(q, k, w, w, inc, interleaved=inter)
    where = torch.tensor([24, 33, 47], device=cuda)
    w[where] = torch.tensor([math.inf, -math.inf, math.inf], dtype=dtype, device=cuda)
    got = rope.qk_norm_rope(q, k, w, w, inc, interleaved=inter)
    for x, c, o in zip((q, k), clean, got):
        want = c.clone()
        want[..., where] = (x[..., where] * w[where].to(torch.float16)).transpose(1, 2)
        assert torch.equal(o, want)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("empty", [dict(batch=0), dict(sequence_length=0), dict(q_heads=0), dict(k_heads=0)],
                         ids=lambda e: next(iter(e)))
def test_weight_gradients_without_rows(cuda, capi, empty, f32):
    """The C entry's sum over no rows is zero, and the other side's is its own."""
    from test_qk_rope_cpu import Args

    dt = torch.float32 if f32 else torch.float16
    sizes = {**dict(batch=2, sequence_length=3, q_heads=2, k_heads=2), **empty}
    ones = torch.ones(2, 3, 2, 64, dtype=torch.float16, device=cuda)
    w = torch.ones(64, dtype=dt, device=cuda)
    dq, dk, = torch.empty_like(ones), torch.empty_like(ones)
    dqw, dkw = (torch.full((64,), 7.0, dtype=dt, device=cuda) for _ in range(2))
    lib = capi.lib
    lib.spline_hip_qk_norm_rope_bwd_bytes.restype = ctypes.c_int64
    ws = torch.full((lib.spline_hip_qk_norm_rope_bwd_bytes(ctypes.c_int64(64)) // 4,), math.nan, device=cuda)
    strides = (ctypes.c_int64 * 3)(384, 128, 64)
    a = Args(q_out=dq.data_ptr(), k_out=dk.data_ptr(), q=ones.data_ptr(), k=ones.data_ptr(), q_weight=w.data_ptr(),
             k_weight=w.data_ptr(), axes=1, head_dim=64, rotary_dim=0, position_bytes=4, weight_f32=int(f32),
             dq_out=ones.data_ptr(), dk_out=ones.data_ptr(), dq_weight=dqw.data_ptr(), dk_weight=dkw.data_ptr(),
             dw_workspace=ws.data_ptr(), eps=0.0, **sizes,
             **{n: strides for n in ("q_strides", "k_strides", "q_out_strides", "k_out_strides", "dq_out_strides",
                                     "dk_out_strides")})
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.launch_qk_norm_rope_bwd_fp16(ctypes.byref(a), stream) == 0
    torch.cuda.synchronize()
    rows = sizes["batch"] * sizes["sequence_length"]
    for got, heads in ((dqw, sizes["q_heads"]), (dkw, sizes["k_heads"])):  # x r = 1 for every row, dy = 1
        assert bool((got.double() - rows * heads).abs().max() <= rows * heads * 2.0 ** -20)
