"""Host side of the shared-prefix attention: what its entry points refuse before
they launch anything, and its workspace (runs without a GPU)."""

import ctypes

import pytest
import torch

import capi_helpers


class Args(ctypes.Structure):
    """spline_hip_shared_prefix."""

    _fields_ = ([(n, ctypes.c_void_p) for n in (
        "out", "lse", "q", "prefix_k", "prefix_v", "suffix_k", "suffix_v", "suffix_lens", "workspace")]
        + [(n, ctypes.c_int64) for n in ("batch", "tokens", "q_heads", "kv_heads", "prefix", "suffix", "head_dim")]
        + [("q_strides", ctypes.c_int64 * 3), ("prefix_k_strides", ctypes.c_int64 * 2),
           ("prefix_v_strides", ctypes.c_int64 * 2), ("suffix_k_strides", ctypes.c_int64 * 3),
           ("suffix_v_strides", ctypes.c_int64 * 3), ("mode", ctypes.c_int32), ("scale", ctypes.c_float),
           ("cap", ctypes.c_float)])


def _args(**changes):
    a = Args(**{n: 4096 for n in ("out", "lse", "q", "prefix_k", "prefix_v", "suffix_k", "suffix_v", "suffix_lens",
                                  "workspace")},
             batch=2, tokens=1, q_heads=8, kv_heads=2, prefix=100, suffix=50, head_dim=128, mode=0, scale=0.1, cap=30.0)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(capi_helpers.LIB)
    lib.spline_hip_shared_prefix_workspace_bytes.restype = ctypes.c_int64
    return lib


SIZES = [dict(batch=-1), dict(tokens=-1), dict(q_heads=0), dict(kv_heads=0), dict(q_heads=7), dict(head_dim=96),
         dict(prefix=-1), dict(suffix=-1), dict(prefix=2 ** 31), dict(suffix=2 ** 31), dict(tokens=2 ** 20),
         dict(q_heads=2 ** 17, kv_heads=2 ** 17), dict(batch=2 ** 31), dict(batch=2 ** 40), dict(batch=2 ** 28, q_heads=8)]
BAD = SIZES + [
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(mode=1), dict(mode=5),
    dict(mode=-1), dict(mode=3, cap=0.0), dict(mode=3, cap=float("inf")), dict(q=None), dict(out=None), dict(q=4104),
    dict(out=4104), dict(lse=4098), dict(prefix_k=None), dict(prefix_v=4104), dict(suffix_k=None), dict(suffix_v=4104),
    dict(suffix_lens=None), dict(suffix_lens=4098), dict(workspace=None), dict(workspace=4104),
    dict(q_strides=(ctypes.c_int64 * 3)(8, 8, 4)), dict(prefix_v_strides=(ctypes.c_int64 * 2)(4, 8)),
    dict(suffix_k_strides=(ctypes.c_int64 * 3)(-8, 8, 8)),
]


@pytest.mark.parametrize("name", ["launch_shared_prefix_attention_bf16", "launch_shared_prefix_attention_fp16"])
@pytest.mark.parametrize("bad", BAD, ids=lambda b: "-".join(f"{k}-{v}" for k, v in b.items() if "strides" not in k))
def test_refuses(lib, name, bad):
    assert getattr(lib, name)(ctypes.byref(_args(**bad)), None) == 1


def test_d4_softcap_takes_bf16(lib):
    assert lib.launch_shared_prefix_attention_fp16(ctypes.byref(_args(mode=4)), None) == 1
    assert lib.launch_shared_prefix_attention_bf16(ctypes.byref(_args(mode=4, cap=0.0)), None) == 1


def test_nothing_to_do(lib):
    for empty in (dict(batch=0), dict(tokens=0)):
        assert lib.launch_shared_prefix_attention_bf16(ctypes.byref(_args(**empty)), None) == 0
        assert lib.spline_hip_shared_prefix_workspace_bytes(ctypes.byref(_args(**empty))) == 0
    assert lib.launch_shared_prefix_attention_bf16(None, None) == 1


def test_workspace(lib):
    """Whole parts of every row's O, maximum and sum; none without keys; the
    sizes that are refused have none."""
    size = lambda **c: lib.spline_hip_shared_prefix_workspace_bytes(ctypes.byref(_args(**c)))  # noqa: E731
    rows = 2 * 8
    for c in (dict(), dict(prefix=100000), dict(suffix=100000), dict(prefix=0), dict(suffix=0)):
        assert size(**c) > 0 and size(**c) % (rows * 130 * 4) == 0
    assert size(prefix=0, suffix=0) == 0
    for bad in SIZES:
        assert size(**bad) == -1, bad


def test_python_refuses_host_tensors():
    from sfu_repro import fa4_runtime

    q, k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa4_runtime.flash_attn_shared_prefix(q, k, k, k[None], k[None], torch.zeros(1, dtype=torch.int32))


def test_limits(lib):
    """2^30 keys and 2^14 tokens: where a part ends is counted in 32 bits."""
    size = lambda **c: lib.spline_hip_shared_prefix_workspace_bytes(ctypes.byref(_args(**c)))
    one = dict(batch=1, q_heads=1, kv_heads=1, head_dim=64)
    for most in (dict(prefix=2 ** 30), dict(suffix=2 ** 30), dict(tokens=2 ** 14)):
        assert size(**one, **most) > 0
        assert size(**one, **{k: v + 1 for k, v in most.items()}) == -1


def test_forward_mode_is_refused():
    """A dual tensor does not require gradients; its tangent is not dropped."""
    from torch.autograd import forward_ad
    from sfu_repro import fa4_runtime

    q, k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    operands = [q, k, k, k[None], k[None]]
    with torch.no_grad(), forward_ad.dual_level():
        for i, t in enumerate(operands):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="flash_attn_shared_prefix has no forward-mode derivative"):
                fa4_runtime.flash_attn_shared_prefix(*operands[:i], dual, *operands[i + 1:],
                                                     torch.zeros(1, dtype=torch.int32))
