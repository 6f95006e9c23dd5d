"""How many workgroups the 4-bit attention's keys are dealt to, told by its workspace (CPU): as many as the chip holds at once."""
import ctypes as C

import pytest

from roost_amd import abi
from test_f4_abi import BF16, F4, I32, U8, _span, ctx  # noqa: F401


def _places(kernels, ctx, q_heads, kv_heads, dim, q_len):  # noqa: F811
    """Two partial places of `most` rows, each head_dim sums, a maximum and a sum, for each workgroup."""
    batch, blocks, page = 64, 1000, 64
    p = abi.new(abi.PagedAttentionF4Params)
    values = kv_heads * page * dim
    c = p.cache
    c.kv_heads, c.head_dim, c.page_size = kv_heads, dim, page
    c.k, c.v = _span(1 << 40, values, F4), _span(2 << 40, values, F4)
    c.k_scales, c.v_scales = _span(3 << 40, values // 32, U8), _span(4 << 40, values // 32, U8)
    p.batch, p.tokens, p.q_heads, p.window_left, p.causal = batch, batch * q_len, q_heads, -1, 1
    n = p.tokens * q_heads * dim
    p.q, p.output, p.cu_seqlens = _span(5 << 40, n, BF16), _span(6 << 40, n, BF16), _span(7 << 40, batch + 1, I32)
    p.block_tables, p.kv_lens = _span(8 << 40, batch * blocks, I32), _span(9 << 40, batch, I32)
    p.table_rows, p.max_blocks, p.max_q_len, p.max_kv_len = batch, blocks, q_len, blocks * page
    sizes = abi.new(abi.WorkspaceSizes)
    assert kernels.dll.roost_amd_paged_attention_f4_workspace(ctx, C.addressof(p), C.addressof(sizes)) == abi.OK
    group = q_heads // kv_heads
    few = max(32 if dim < 256 and (group > 16 or 16 < q_len * group <= 32) else 16, group)
    row = (dim + 2) * 4
    parts, rest = divmod(sizes.device_bytes - 4 * (batch + 1), 2 * (few // group) * group * row)
    assert rest == 0
    return parts


@pytest.mark.parametrize("q_heads,kv_heads,dim,q_len,a_cu", [
    (32, 8, 64, 1, 4), (32, 8, 128, 1, 3), (32, 8, 256, 1, 2),   # one tile of 16 rows
    (32, 8, 64, 8, 2), (32, 8, 128, 8, 2), (32, 8, 128, 5, 2),   # two tiles: drafts
    (64, 2, 64, 1, 2), (64, 2, 128, 1, 2), (34, 2, 128, 1, 2),   # two tiles: groups above 16
    (64, 2, 256, 1, 2)])
def test_keys_are_dealt_to_what_the_chip_holds(kernels, ctx, q_heads, kv_heads, dim, q_len, a_cu):  # noqa: F811
    cus = _places(kernels, ctx, 32, 8, 256, 1) // 2  # head_dim 256: two workgroups a CU
    assert cus >= 64 and _places(kernels, ctx, q_heads, kv_heads, dim, q_len) == a_cu * cus
