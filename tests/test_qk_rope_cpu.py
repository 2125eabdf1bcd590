"""Host side of the head norm and the rotations: the builders, and what the
entry points refuse before they launch anything (runs without a GPU)."""

import ctypes
import math

import pytest
import torch

import capi_helpers
import qk_rope_reference as ref


class Args(ctypes.Structure):
    """spline_hip_qk_rope."""

    _fields_ = ([(n, ctypes.c_void_p) for n in (
        "q_out", "k_out", "q", "k", "q_weight", "k_weight", "phase_increments", "positions", "frequency_axes")]
        + [(n, ctypes.c_int64) for n in (
            "axes", "batch", "sequence_length", "q_heads", "k_heads", "head_dim", "rotary_dim")]
        + [(n, ctypes.c_int64 * 3) for n in (
            "q_strides", "k_strides", "q_out_strides", "k_out_strides", "position_strides")]
        + [(n, ctypes.c_int32) for n in ("position_bytes", "weight_f32", "interleaved")] + [("eps", ctypes.c_float)]
        + [(n, ctypes.c_void_p) for n in ("dq_out", "dk_out")]
        + [(n, ctypes.c_int64 * 3) for n in ("dq_out_strides", "dk_out_strides")]
        + [(n, ctypes.c_void_p) for n in ("dq_weight", "dk_weight", "dw_workspace")])


def _args(**changes):
    """Arguments with nothing wrong but an empty batch; the addresses are never used."""
    a = Args(q_out=4096, k_out=4096, q=4096, k=4096, phase_increments=4096, axes=1, batch=0, sequence_length=4,
             q_heads=2, k_heads=1, head_dim=64, rotary_dim=64, position_bytes=8, dq_out=4096, dk_out=4096)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(capi_helpers.LIB)


BAD = [
    dict(batch=-1), dict(sequence_length=-1), dict(q_heads=-1), dict(k_heads=-1), dict(head_dim=0),
    dict(head_dim=60), dict(head_dim=264), dict(rotary_dim=72), dict(rotary_dim=12), dict(rotary_dim=-8),
    dict(q_heads=65537),
    dict(batch=2 ** 31, sequence_length=1), dict(batch=2 ** 16, sequence_length=2 ** 16),
    dict(batch=2, phase_increments=None), dict(batch=2, phase_increments=4098), dict(batch=2, position_bytes=2),
    dict(batch=2, positions=4100), dict(batch=2, frequency_axes=4096), dict(batch=2, q=None), dict(batch=2, k_out=None),
    dict(batch=2, q=4098), dict(batch=2, k=4100), dict(batch=2, q_weight=4097),
    dict(batch=2, q_strides=(ctypes.c_int64 * 3)(2, 64, 64)), dict(batch=2, k_out_strides=(ctypes.c_int64 * 3)(64, 64, 3)),
    dict(batch=2, positions=4096, frequency_axes=4096, axes=0),
]


@pytest.mark.parametrize("name", ["launch_qk_norm_rope_fp16", "launch_qk_norm_rope_bf16", "launch_qk_norm_rope_bwd_fp16",
                                  "launch_qk_norm_rope_bwd_bf16"])
@pytest.mark.parametrize("bad", BAD, ids=lambda b: "-".join(b))
def test_refuses(lib, name, bad):
    assert getattr(lib, name)(ctypes.byref(_args(**bad)), None) == 1


@pytest.mark.parametrize("bad", [b for b in BAD if "q_weight" not in b], ids=lambda b: "-".join(b))
def test_axes_refuses(lib, bad):
    for inverse in (0, 1):
        assert lib.launch_rope_axes_bf16(ctypes.byref(_args(**bad)), inverse, None) == 1


def test_backward_refuses(lib):
    for bad in (dict(dq_out=None), dict(dk_out=4100), dict(q_weight=4096), dict(q_weight=4096, dq_weight=4096),
                dict(q_weight=4096, dw_workspace=4096)):
        assert lib.launch_qk_norm_rope_bwd_bf16(ctypes.byref(_args(batch=2, **bad)), None) == 1
    assert lib.launch_qk_norm_rope_bf16(None, None) == 1


def test_nothing_to_do(lib):
    for empty in (dict(), dict(batch=3, sequence_length=0), dict(batch=3, q_heads=0, k_heads=0)):
        for name in ("launch_qk_norm_rope_fp16", "launch_qk_norm_rope_bwd_bf16"):
            assert getattr(lib, name)(ctypes.byref(_args(**empty)), None) == 0


def test_python_refuses_host_tensors():
    from sfu_repro import rope

    q = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        rope.qk_norm_rope(q, q, None, None, rope.phase_increments(64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        rope.rope_axes(q, q, rope.phase_increments(64), torch.zeros(2, 1, 2, dtype=torch.int64),
                       rope.axis_sections((16, 16)))


def test_phase_increments():
    from sfu_repro import rope

    inc = rope.phase_increments(128, 500000.0)
    freq = 500000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    assert inc.dtype == torch.int32 and inc.numel() == 64
    # half a unit of 2^-32 turns
    assert float((inc.double() * (2 * math.pi / 2 ** 32) - freq).abs().max()) <= math.pi / 2 ** 32 + 1e-15
    assert rope.phase_increments(0).numel() == 0
    with pytest.raises(ValueError, match="even"):
        rope.phase_increments(7)


def test_axis_sections():
    from sfu_repro import rope

    assert rope.axis_sections((2, 0, 3)).tolist() == [0, 0, 2, 2, 2]
    for bad in ((), (1, -1)):
        with pytest.raises(ValueError, match="sections"):
            rope.axis_sections(bad)


def test_reference_angles_are_exact():
    """The reference's modular product, against Python's integers."""
    g = torch.Generator().manual_seed(0)
    pos = torch.randint(-2 ** 40, 2 ** 40, (1, 50), generator=g)
    inc = torch.randint(-2 ** 31, 2 ** 31, (4,), generator=g).to(torch.int32)
    got = ref.angles(inc, pos, None, 1, 50)[0, :, 0] * (2 ** 32 / (2 * math.pi))
    want = [[p * (i % 2 ** 32) % 2 ** 32 for i in inc.tolist()] for p in pos[0].tolist()]
    assert torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=0, atol=1e-5)


@pytest.mark.parametrize("interleaved", [True, False])
def test_reference_gradients(interleaved):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 3, 2, 16, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(16, generator=g, dtype=torch.float64, requires_grad=True)
    theta = torch.randn(1, 3, 1, 4, generator=g, dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda a, b: ref.heads_out(a, b, theta, 1e-6, interleaved, True), (x, w))


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    """A dual tensor does not require gradients; its tangent is not dropped."""
    from torch.autograd import forward_ad
    from sfu_repro import rope

    q, inc = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16), rope.phase_increments(64)
    w, pos = torch.ones(64), torch.zeros(2, 1, 2, dtype=torch.int64)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual, dual_w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (q, w))
        for args in ((dual, q, None, None), (q, dual, None, None), (q, q, dual_w, None), (q, q, w, dual_w)):
            with pytest.raises(RuntimeError, match="qk_norm_rope has no forward-mode derivative"):
                rope.qk_norm_rope(*args, inc)
        for args in ((dual, q), (q, dual)):
            with pytest.raises(RuntimeError, match="rope_axes has no forward-mode derivative"):
                rope.rope_axes(*args, inc, pos, rope.axis_sections((16, 16)))


def test_forward_mode_of_the_gradients_is_refused():
    import spline_ops
    from torch.autograd import forward_ad
    from sfu_repro import rope

    q, inc = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16), rope.phase_increments(64)
    pos = torch.zeros(2, 1, 2, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for dq, dk in ((dual, q), (q, dual)):
            with pytest.raises(RuntimeError, match="qk_norm_rope has no forward-mode derivative"):
                spline_ops.qk_norm_rope_bwd(q, q, None, None, inc, None, None, dq, dk, 1e-6, True)
            with pytest.raises(RuntimeError, match="rope_axes has no forward-mode derivative"):
                spline_ops.rope_axes_bwd(dq, dk, inc, pos, rope.axis_sections((16, 16)), True)
