"""Head norm at the ends of what its operands hold: weights that are no numbers,
sides and batches without a row; and captured backward passes beside eager graphs."""

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


def _captured_step(cuda):
    from sfu_repro import rope

    g = torch.Generator(device=cuda).manual_seed(31)
    q, k = (torch.randn(2, 30, h, 64, generator=g, device=cuda).half().requires_grad_(True) for h in (4, 2))
    w = torch.ones(64, device=cuda).requires_grad_(True)
    inc = rope.phase_increments(64).to(cuda)
    d = [torch.randn(2, h, 30, 64, generator=g, device=cuda).half() for h in (4, 2)]
    return q, k, w, d, lambda *leaves: rope.qk_norm_rope(leaves[0], leaves[1], leaves[2], leaves[2], inc)


def test_capture_of_gradients_that_other_leaves_do_not_take(cuda):
    """An eager graph of leaves that the captured pass does not ask for is no
    reason to refuse it: of a subset of them, or of activations alone."""
    q, k, w, d, call = _captured_step(cuda)
    alive = call(q, k, torch.ones_like(w))  # q and k, not w
    want = torch.autograd.grad(call(q, k, w), w, d)[0]
    scaled = (q.detach() * 0.5).requires_grad_(True)
    want_q = torch.autograd.grad(call(scaled, k, w), scaled, d)[0]
    del scaled
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(call(q, k, w), w, d)[0]
        x = q * 0.5
        held_q = torch.autograd.grad(call(x, k, w), x, d)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(held_q, want_q)
    with pytest.raises(RuntimeError, match="capture on its stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(call(q, k, w), [w, q], d)
    del alive


def test_capture_on_the_stream_of_the_eager_graph(cuda):
    q, k, w, d, call = _captured_step(cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        alive = call(q, k, w)
        want = torch.autograd.grad(alive, [q, k, w], d, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = torch.autograd.grad(call(q, k, w), [q, k, w], d)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    del alive
