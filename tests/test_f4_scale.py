"""The 4-bit attention's sm_scale at the end of its range."""
import ctypes as C

import pytest
import torch

from roost_amd import abi
from test_f4_abi import NOT, SMALL, _attention, ctx  # noqa: F401


@pytest.mark.parametrize("scale,want", [(2.0 ** 126, SMALL), (2.0 ** 126 * (1 + 2.0 ** -23), NOT), (3e38, NOT)])
def test_scales_whose_product_with_log2_e_passes_f32(kernels, ctx, scale, want):  # noqa: F811
    """In that unit every score of 0 would be 0 times infinity. SMALL: admitted, and told of the workspace that is not there."""
    p = _attention()
    p.sm_scale, p.max_kv_len = scale, 4096
    assert kernels.dll.roost_amd_paged_attention_f4_run(ctx, C.addressof(p), None, None) == want, kernels.last_error()
    sizes = abi.new(abi.WorkspaceSizes)
    status = kernels.dll.roost_amd_paged_attention_f4_workspace(ctx, C.addressof(p), C.addressof(sizes))
    assert status == (NOT if want == NOT else abi.OK)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** 126, 2.0 ** -126, 2.0 ** -149])
def test_scores_of_zero_at_any_scale(session, scale):
    import f4_cases as fc

    a = fc.Attention(93, [(1, 300), (40, 90)], dim=128, scale=scale)
    a.q.zero_()
    a.run(session)
    a.check()
    assert torch.isfinite(a.lse).all()
