"""Score programs that the serving attentions are not built with (refused ahead of any launch)."""

import pytest
import torch


@pytest.mark.parametrize("program", [
    dict(sigmoid_attention=True), dict(sigmoid_attention=True, sigmoid_poly_backend="device"),
    dict(sigmoid_attention=True, sigmoid_poly_backend="device", sigmoid_degree=2),
    dict(sigmoid_attention=True, sigmoid_sfu_res=16), dict(exp2_emu_freq=16)], ids=str)
def test_a_program_that_is_not_built_is_named(program):
    from sfu_repro import fa4_runtime

    q, k = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    cache, n = torch.zeros(1, 2, 2, 16 * 34, dtype=torch.uint8), torch.ones(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError, match="over 4-bit pages is built with"):
        fa4_runtime.flash_attn_paged_fp4(q, cache, n[None], n, **program)
    with pytest.raises(NotImplementedError, match="shared-prefix attention is built with"):
        fa4_runtime.flash_attn_shared_prefix(q, k, k, k[None], k[None], n, **program)
