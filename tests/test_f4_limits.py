"""What the 4-bit attention's launches can hold, and what the Python mirrors of the cache and page calls refuse (CPU)."""
import ctypes as C

import pytest
import torch

import roost_amd
from roost_amd import abi
from test_f4_abi import BF16, I32, NOT, SMALL, _cache, _span, ctx  # noqa: F401


def _wide(batch, tokens, q_heads, kv_heads):
    p = abi.new(abi.PagedAttentionF4Params)
    _cache(p)
    c, page = p.cache, p.cache.page_size * p.cache.head_dim * kv_heads
    c.kv_heads = kv_heads
    c.k.length = c.v.length = page
    c.k_scales.length = c.v_scales.length = page // 32
    c.k.address, c.v.address, c.k_scales.address, c.v_scales.address = (x << 40 for x in (1, 2, 3, 4))
    p.batch, p.tokens, p.q_heads, p.window_left, p.causal = batch, tokens, q_heads, -1, 1
    n = tokens * q_heads * c.head_dim
    p.q, p.output, p.cu_seqlens = _span(5 << 40, n, BF16), _span(6 << 40, n, BF16), _span(7 << 40, batch + 1, I32)
    p.block_tables, p.kv_lens = _span(8 << 40, batch, I32), _span(9 << 40, batch, I32)
    p.table_rows, p.max_blocks = batch, 1
    return p


@pytest.mark.parametrize("batch,tokens,q_len,q_heads,kv_heads,want", [
    (65535, 65535, 1, 1024, 1024, NOT),      # a workgroup for each sequence and KV head: 2^26 of them
    (65535, 1 << 20, 0, 1024, 1024, NOT),    # tiles of up to 61,680 sequences in each head
    (700, 700, 1, 1024, 1024, SMALL),        # dealt: few workgroups, and a workspace
])
def test_launches(kernels, ctx, batch, tokens, q_len, q_heads, kv_heads, want):  # noqa: F811
    p = _wide(batch, tokens, q_heads, kv_heads)
    p.max_q_len = q_len
    assert kernels.dll.roost_amd_paged_attention_f4_run(ctx, C.addressof(p), None, None) == want, kernels.last_error()
    sizes = abi.new(abi.WorkspaceSizes)
    status = kernels.dll.roost_amd_paged_attention_f4_workspace(ctx, C.addressof(p), C.addressof(sizes))
    assert status == (NOT if want == NOT else abi.OK) and (sizes.device_bytes > 0) == (want == SMALL)


def test_a_large_batch_needs_no_workspace(kernels, ctx):  # noqa: F811
    p = _wide(65535, 65535, 255, 255)
    p.max_q_len = 1
    sizes = abi.new(abi.WorkspaceSizes)
    assert kernels.dll.roost_amd_paged_attention_f4_workspace(ctx, C.addressof(p), C.addressof(sizes)) == abi.OK
    assert sizes.device_bytes == 0


def test_python_checks():
    """Shapes, strides, types and devices that the records cannot carry."""
    cache = roost_amd.cache_f4(3, 2, 16, 64, device="cpu")
    assert [tuple(t.shape) for t in cache] == [(3, 2, 16, 32), (3, 2, 2, 16)] * 2
    c = roost_amd._cache_f4(cache)
    assert (c.kv_heads, c.head_dim, c.page_size, c.k.length, c.v_scales.length) == (2, 64, 16, 3 * 2 * 16 * 64, 3 * 2 * 2 * 16)
    assert c.k.dtype == abi.DTYPE_F4E2M1
    for i, bad in ((0, cache.k[0]), (1, cache.k_scales.transpose(2, 3)), (2, cache.v[:2]), (3, cache.v_scales.int()),
                   (0, cache.k.transpose(0, 1))):
        with pytest.raises(ValueError, match="cache"):
            roost_amd._cache_f4(tuple(bad if j == i else t for j, t in enumerate(cache)))

    rows = torch.zeros(5, 6, 64)
    assert roost_amd._token_heads(rows[:, 2:4], "k", 5, 2, 64)[1] == 6 * 64
    assert roost_amd._token_heads(rows[:1, :2], "k", 1, 2, 64)[1] == 2 * 64
    for bad in (rows, rows[:, ::3], rows[..., ::2], rows[:1, :2].expand(5, 2, 64), rows[:4, :2]):
        with pytest.raises(ValueError, match="k: "):
            roost_amd._token_heads(bad, "k", 5, 2, 64)

    found, pages = roost_amd._pools([torch.zeros(2, 7, 4, 4), torch.zeros(9, 7, 32, dtype=torch.uint8)[:3]])
    assert pages == 7 and (found[0].page_bytes, found[0].layers, found[0].layer_bytes) == (64, 2, 7 * 64)
    assert (found[1].page_bytes, found[1].layers, found[1].layer_bytes) == (32, 3, 7 * 32)
    for bad in ([], [torch.zeros(2, 7, 4), torch.zeros(2, 6, 4)], [torch.zeros(7)], [torch.zeros(0, 7, 4)],
                [torch.zeros(2, 7, 8)[..., :4]], [torch.zeros(7, 2, 4).transpose(0, 1)]):
        with pytest.raises(ValueError, match="pool"):
            roost_amd._pools(bad)

    i32 = torch.zeros(3, dtype=torch.int32)
    tables = dict(block_tables=torch.zeros(3, 4, dtype=torch.int32), lengths=i32, refs=i32, page_size=16)
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: roost_amd.cache_f4_params(q, q, cache, i32),
                 lambda: roost_amd.paged_attention_f4_params(q, q, cache, i32, block_tables=tables["block_tables"], kv_lens=i32),
                 lambda: roost_amd.cache_copy_params([rows], i32.view(-1, 1)),
                 lambda: roost_amd.cache_free_params(i32, **tables)):
        with pytest.raises(ValueError, match="tensors of one call are on"):
            call()
    for half in (dict(), dict(block_tables=i32), dict(kv_lens=i32), dict(kv_indptr=i32, kv_indices=i32),
                 dict(block_tables=i32, kv_lens=i32, kv_indptr=i32, kv_indices=i32, kv_last_page_len=i32),
                 dict(kv_indptr=i32, kv_indices=i32, kv_last_page_len=i32, sequences=i32)):
        with pytest.raises(ValueError, match="tables: "):
            roost_amd.paged_attention_f4_params(q, q, cache, i32, **half)
