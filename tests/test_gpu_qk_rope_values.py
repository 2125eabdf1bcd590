"""Head norm with weights at the ends of what their type holds."""

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
