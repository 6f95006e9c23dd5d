"""The 4-bit cache's calls and the page calls without a GPU: record layouts, typed refusals (each before any launch), the
format's definition and the definitions of the page calls."""
import ctypes as C

import pytest
import torch

import f4_cases as fc
from roost_amd import abi

BF16, F16, F32, F4, U8, I32, I64 = (abi.DTYPE_BF16, abi.DTYPE_F16, abi.DTYPE_F32, abi.DTYPE_F4E2M1, abi.DTYPE_U8, abi.DTYPE_I32,
                                    abi.DTYPE_I64)
BAD, NOT, OLD, SMALL = abi.INVALID_ARGUMENT, abi.UNSUPPORTED, abi.ABI_MISMATCH, abi.WORKSPACE_TOO_SMALL


def _span(address, n, dtype):
    s = abi.DeviceSpan()
    s.address, s.length, s.dtype = address, n, dtype
    return s


@pytest.fixture()
def ctx(kernels):
    c = kernels.create_context(0)
    yield c
    kernels.destroy_context(c)


def _set(p, path, value):
    *outer, name = path.split(".")
    for o in outer:
        p = getattr(p, o)
    setattr(p, name, value)


def test_layouts():
    sizes = {"RoostAmdCacheF4": 112, "RoostAmdCacheF4Params": 208, "RoostAmdPagedAttentionF4Params": 360, "RoostAmdPagePool": 32,
             "RoostAmdCacheCopyParams": 56, "RoostAmdCachePagesParams": 208}
    for name, size in sizes.items():
        assert C.sizeof(abi.EXTENSION_STRUCTS[name]) == size, name
    assert (abi.CacheF4.kv_heads.offset, abi.CacheF4Params.cache.offset, abi.CacheF4Params.tokens.offset) == (96, 56, 192)
    p = abi.PagedAttentionF4Params
    assert (p.cache.offset, p.cu_seqlens.offset, p.batch.offset, p.sm_scale.offset, p.causal.offset) == (80, 192, 312, 344, 356)
    assert (abi.CacheCopyParams.pairs.offset, abi.CachePagesParams.block_tables.offset, abi.CachePagesParams.sequences.offset) == \
        (24, 24, 192)


# ---- the cache -----------------------------------------------------------------------------------------------------------

PAGE = 2 * 16 * 128  # values of a page of 2 heads, 16 tokens, 128 dims


def _cache(p, pages=4):
    p.cache.k, p.cache.v = _span(0x1000000, pages * PAGE, F4), _span(0x2000000, pages * PAGE, F4)
    p.cache.k_scales, p.cache.v_scales = _span(0x3000000, pages * PAGE // 32, U8), _span(0x4000000, pages * PAGE // 32, U8)
    p.cache.kv_heads, p.cache.head_dim, p.cache.page_size = 2, 128, 16


def _write():
    p = abi.new(abi.CacheF4Params)
    _cache(p)
    p.tokens, p.k_stride, p.v_stride = 5, 768, 768
    p.k, p.v = _span(0x100000, 4 * 768 + 256, BF16), _span(0x100200, 4 * 768 + 256, BF16)  # columns of one projection
    p.slot_mapping = _span(0x500000, 5, I64)
    return p


CACHE_REFUSALS = [
    ("cache.reserved0", 1, BAD), ("cache.kv_heads", 0, NOT), ("cache.kv_heads", 1025, NOT), ("cache.head_dim", 96, NOT),
    ("cache.head_dim", 512, NOT), ("cache.page_size", 8, NOT), ("cache.page_size", 24, NOT), ("cache.page_size", 2048, NOT),
    ("cache.k.dtype", U8, BAD), ("cache.v_scales.dtype", F4, BAD), ("cache.k.length", PAGE - 1, BAD),
    ("cache.v_scales.length", PAGE // 32 - 1, BAD), ("cache.v.address", None, BAD), ("cache.k_scales.address", 0x3000008, BAD),
    ("cache.k.reserved0", 7, BAD)]


@pytest.mark.parametrize("call", ["write", "read"])
@pytest.mark.parametrize("field,value,want", CACHE_REFUSALS + [
    ("struct_size", 100, OLD), ("abi_minor", 99, OLD), ("reserved0", 1, BAD), ("k.dtype", abi.DTYPE_F8E4M3, NOT), ("k.dtype", F32, BAD),
    ("k.length", 4 * 768 + 255, BAD), ("v.address", None, BAD), ("k.address", 0x100008, BAD), ("k_stride", 255, BAD),
    ("v_stride", 772, BAD), ("tokens", 1 << 24, NOT), ("slot_mapping.length", 4, BAD), ("slot_mapping.dtype", I32, BAD),
    ("slot_mapping.address", 0x500004, BAD), ("v.address", 0x1000100, BAD), ("slot_mapping.address", 0x3000000, BAD)])
def test_cache_refusals(kernels, ctx, call, field, value, want):
    run = getattr(kernels.dll, f"roost_amd_cache_{call}_f4_run")
    p = _write()
    _set(p, field, value)
    assert run(ctx, C.addressof(p), None) == want, kernels.last_error()
    assert kernels.last_error()


def test_cache_refusals_of_one_direction(kernels, ctx):
    p = _write()
    p.k.dtype = p.v.dtype = F16
    assert kernels.dll.roost_amd_cache_read_f4_run(ctx, C.addressof(p), None) == NOT
    p = _write()
    p.v = _span(0x100100, 4 * 768 + 256, BF16)  # shares columns with k: two rows to read, but not to write
    assert kernels.dll.roost_amd_cache_read_f4_run(ctx, C.addressof(p), None) == BAD
    p = _write()
    p.cache.v.address = p.cache.k.address       # one span for both: to read, but not to write
    assert kernels.dll.roost_amd_cache_write_f4_run(ctx, C.addressof(p), None) == BAD
    p = _write()
    assert kernels.dll.roost_amd_cache_write_f4_run(None, C.addressof(p), None) == BAD
    assert kernels.dll.roost_amd_cache_write_f4_run(ctx, None, None) == BAD
    p.tokens = 0
    assert kernels.dll.roost_amd_cache_write_f4_run(ctx, C.addressof(p), None) == abi.OK


# ---- attention ------------------------------------------------------------------------------------------------------------

def _attention(csr=False):
    p = abi.new(abi.PagedAttentionF4Params)
    _cache(p)
    p.batch, p.tokens, p.q_heads, p.q_stride = 3, 5, 8, 2048
    p.q, p.output = _span(0x100000, 4 * 2048 + 1024, BF16), _span(0x200000, 5 * 1024, BF16)
    p.lse = _span(0x300000, 40, F32)
    p.cu_seqlens, p.window_left, p.causal = _span(0x500000, 4, I32), -1, 1
    if csr:
        p.kv_indptr, p.block_tables, p.kv_lens = _span(0x510000, 4, I32), _span(0x520000, 9, I32), _span(0x530000, 3, I32)
    else:
        p.block_tables, p.kv_lens = _span(0x520000, 6 * 2, I32), _span(0x530000, 6, I32)
        p.sequences, p.table_rows, p.max_blocks = _span(0x540000, 3, I32), 6, 2
    return p


ATTENTION_REFUSALS = CACHE_REFUSALS + [
    ("struct_size", 352, OLD), ("q_heads", 0, NOT), ("q_heads", 7, NOT), ("q_heads", 66, NOT), ("batch", 65536, NOT),
    ("tokens", 1 << 24, NOT), ("q.dtype", F32, NOT), ("output.dtype", F32, NOT), ("causal", 2, BAD), ("window_left", -2, BAD),
    ("window_left", (1 << 30) + 1, BAD), ("sm_scale", -1.0, BAD), ("sm_scale", float("nan"), BAD), ("sm_scale", float("inf"), BAD),
    ("logits_soft_cap", -1.0, BAD), ("logits_soft_cap", float("nan"), BAD), ("q_stride", 1016, BAD), ("q_stride", 2049, BAD),
    ("q.length", 4 * 2048 + 1023, BAD), ("q.address", 0x100008, BAD), ("output.length", 5 * 1024 - 1, BAD),
    ("output.address", 0x200004, BAD), ("lse.length", 39, BAD), ("lse.dtype", BF16, BAD), ("lse.address", 0x300002, BAD),
    ("cu_seqlens.length", 3, BAD), ("cu_seqlens.dtype", I64, BAD), ("kv_lens.address", None, BAD),
    ("output.address", 0x100000, BAD), ("output.address", 0x1000000, BAD), ("lse.address", 0x200010, BAD),
    ("lse.address", 0x520000, BAD)]


@pytest.mark.parametrize("csr", [False, True])
@pytest.mark.parametrize("field,value,want", ATTENTION_REFUSALS)
def test_attention_refusals(kernels, ctx, csr, field, value, want):
    p = _attention(csr)
    _set(p, field, value)
    assert kernels.dll.roost_amd_paged_attention_f4_run(ctx, C.addressof(p), None, None) == want, kernels.last_error()
    sizes = abi.new(abi.WorkspaceSizes)
    assert kernels.dll.roost_amd_paged_attention_f4_workspace(ctx, C.addressof(p), C.addressof(sizes)) == want


@pytest.mark.parametrize("csr,field,value", [
    (False, "max_blocks", 0), (False, "table_rows", 0), (False, "block_tables.length", 11), (False, "kv_lens.length", 5),
    (False, "sequences.length", 2), (False, "table_rows", 7), (True, "max_blocks", 1), (True, "table_rows", 1),
    (True, "kv_indptr.length", 3), (True, "kv_lens.length", 2), (True, "sequences", _span(0x540000, 3, I32)),
    (True, "block_tables.address", None)])
def test_attention_tables(kernels, ctx, csr, field, value):
    p = _attention(csr)
    _set(p, field, value)
    assert kernels.dll.roost_amd_paged_attention_f4_run(ctx, C.addressof(p), None, None) == BAD, kernels.last_error()


def test_attention_without_sequences_needs_a_row_each(kernels, ctx):
    p = _attention()
    p.sequences = abi.DeviceSpan()
    p.table_rows, p.block_tables.length = 2, 4
    assert kernels.dll.roost_amd_paged_attention_f4_run(ctx, C.addressof(p), None, None) == BAD
    assert "sequences" in kernels.last_error()


def test_window_needs_causal(kernels, ctx):
    p = _attention()
    p.window_left, p.causal = 5, 0
    assert kernels.dll.roost_amd_paged_attention_f4_run(ctx, C.addressof(p), None, None) == NOT


def test_attention_workspace(kernels, ctx):
    """Asked for by the record's numbers alone; a call without it is refused, an empty one needs none."""
    p = _attention()
    p.max_kv_len = 4096
    sizes = abi.new(abi.WorkspaceSizes)
    assert kernels.dll.roost_amd_paged_attention_f4_workspace(ctx, C.addressof(p), C.addressof(sizes)) == abi.OK
    assert sizes.device_bytes > 0 and sizes.pinned_host_bytes == 0 and sizes.plan_bytes == 0 and sizes.device_alignment == 256
    run = kernels.dll.roost_amd_paged_attention_f4_run
    assert run(ctx, C.addressof(p), None, None) == SMALL
    ws = abi.new(abi.Workspace)
    ws.device, ws.device_bytes = 0x7000000, sizes.device_bytes - 1
    assert run(ctx, C.addressof(p), C.addressof(ws), None) == SMALL
    ws.device, ws.device_bytes = 0x7000010, sizes.device_bytes
    assert run(ctx, C.addressof(p), C.addressof(ws), None) == SMALL
    for empty in ("tokens", "batch"):
        p = _attention()
        setattr(p, empty, 0)
        assert run(ctx, C.addressof(p), None, None) == abi.OK, kernels.last_error()


# ---- pages ----------------------------------------------------------------------------------------------------------------

def _pool(address=0x10000000, page_bytes=1024, layers=2, layer_bytes=64 * 1024):
    p = abi.PagePool()
    p.address, p.page_bytes, p.layers, p.layer_bytes = address, page_bytes, layers, layer_bytes
    return p


def _copy(*pools):
    p = abi.new(abi.CacheCopyParams)
    p._pools = (abi.PagePool * max(1, len(pools)))(*pools)
    p.pools, p.pool_count, p.pages, p.count = C.addressof(p._pools), len(pools), 64, 3
    p.pairs = _span(0x500000, 6, I32)
    return p


@pytest.mark.parametrize("field,value,want", [
    ("struct_size", 48, OLD), ("reserved0", 1, BAD), ("pages", 0, NOT), ("pages", (4 << 20) + 1, NOT), ("count", 65537, NOT),
    ("pairs.length", 5, BAD), ("pairs.dtype", I64, BAD), ("pairs.address", 0x500004, BAD), ("pairs.address", 0x10000100, BAD),
    ("pools", None, BAD), ("pool_count", 0, BAD), ("pool_count", 17, BAD)])
def test_copy_refusals(kernels, ctx, field, value, want):
    p = _copy(_pool())
    _set(p, field, value)
    assert kernels.dll.roost_amd_cache_copy_run(ctx, C.addressof(p), None, None) == want, kernels.last_error()


@pytest.mark.parametrize("pool,want", [
    (_pool(address=None), BAD), (_pool(address=0x10000008), BAD), (_pool(page_bytes=0), BAD), (_pool(page_bytes=1000), BAD),
    (_pool(layers=0), BAD), (_pool(layer_bytes=63 * 1024), BAD), (_pool(layer_bytes=64 * 1024 + 8), BAD),
    (_pool(page_bytes=(1 << 34) + 16, layers=1), NOT), (_pool(layers=1 << 26), NOT), (_pool(layer_bytes=1 << 41), BAD)])
def test_pool_refusals(kernels, ctx, pool, want):
    p = _copy(pool)
    assert kernels.dll.roost_amd_cache_copy_run(ctx, C.addressof(p), None, None) == want, kernels.last_error()
    p = _pages("fork")
    p._pools[0] = pool
    assert kernels.dll.roost_amd_cache_fork_run(ctx, C.addressof(p), None, None) == want, kernels.last_error()


def test_pools_apart(kernels, ctx):
    p = _copy(_pool(), _pool(address=0x10000000 + 64 * 1024))
    assert kernels.dll.roost_amd_cache_copy_run(ctx, C.addressof(p), None, None) == BAD and "overlap" in kernels.last_error()
    p = _copy(_pool(layer_bytes=1 << 20), _pool(address=0x10000000 + 64 * 1024, layer_bytes=1 << 20))  # layers side by side
    p.count = 0
    assert kernels.dll.roost_amd_cache_copy_run(ctx, C.addressof(p), None, None) == abi.OK, kernels.last_error()


def test_copy_workspace(kernels, ctx):
    """Few pairs need none; more than 1,024 a bitmap or three of the pages."""
    sizes = abi.new(abi.WorkspaceSizes)
    p = _copy(_pool())
    p.count, p.pairs.length = 1024, 2048
    assert kernels.dll.roost_amd_cache_copy_workspace(ctx, C.addressof(p), C.addressof(sizes)) == abi.OK
    assert sizes.device_bytes == 0
    p.count, p.pairs.length = 1025, 2050
    assert kernels.dll.roost_amd_cache_copy_workspace(ctx, C.addressof(p), C.addressof(sizes)) == abi.OK
    assert sizes.device_bytes >= 3 * 64 // 8
    assert kernels.dll.roost_amd_cache_copy_run(ctx, C.addressof(p), None, None) == SMALL


CALLS = ["fork", "grow", "free", "compact"]


def _pages(call):
    p = abi.new(abi.CachePagesParams)
    p._pools = (abi.PagePool * 1)(_pool())
    if call in ("fork", "compact"):
        p.pools, p.pool_count = C.addressof(p._pools), 1
    p.sequences, p.max_blocks, p.pages, p.page_size = 6, 5, 64, 16
    p.block_tables, p.lengths, p.refs = _span(0x500000, 30, I32), _span(0x510000, 6, I32), _span(0x520000, 64, I32)
    if call != "compact":
        p.count, p.requests = 3, _span(0x530000, 6, I32)
    if call == "grow":
        p.cu_seqlens, p.slot_mapping = _span(0x540000, 4, I32), _span(0x550000, 20, I64)
    if call != "free":
        p.status = _span(0x560000, 3, I32)
    return p


def _run(kernels, ctx, call, p):
    fn = getattr(kernels.dll, f"roost_amd_cache_{call}_run")
    return fn(ctx, C.addressof(p), None) if call == "free" else fn(ctx, C.addressof(p), None, None)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("field,value,want", [
    ("struct_size", 200, OLD), ("sequences", 0, NOT), ("max_blocks", 0, NOT), ("sequences", 1 << 30, NOT), ("pages", 0, NOT),
    ("pages", (4 << 20) + 1, NOT), ("page_size", 24, NOT), ("page_size", 0, NOT), ("count", 1025, NOT),
    ("block_tables.length", 29, BAD), ("lengths.length", 5, BAD), ("refs.length", 63, BAD), ("refs.dtype", I64, BAD),
    ("lengths.address", None, BAD), ("refs.address", 0x520002, BAD), ("refs.address", 0x500008, BAD), ("lengths.address", 0x520000, BAD)])
def test_table_refusals(kernels, ctx, call, field, value, want):
    p = _pages(call)
    _set(p, field, value)
    assert _run(kernels, ctx, call, p) == want, kernels.last_error()


@pytest.mark.parametrize("call,field,value", [
    ("fork", "requests.length", 5), ("grow", "requests.length", 2), ("free", "requests.dtype", I64), ("fork", "pools", None),
    ("compact", "pool_count", 0), ("grow", "cu_seqlens.length", 3), ("grow", "cu_seqlens.address", None),
    ("grow", "slot_mapping.address", None), ("grow", "slot_mapping.dtype", I32), ("grow", "slot_mapping.address", 0x550004),
    ("fork", "status.length", 2), ("compact", "status.dtype", I64), ("fork", "requests.address", 0x500000),
    ("grow", "cu_seqlens.address", 0x550000), ("free", "requests.address", 0x510000), ("fork", "status.address", 0x520000),
    ("compact", "refs.address", 0x10000000)])
def test_request_refusals(kernels, ctx, call, field, value):
    p = _pages(call)
    _set(p, field, value)
    assert _run(kernels, ctx, call, p) == BAD, kernels.last_error()


def test_pages_workspace(kernels, ctx):
    sizes = abi.new(abi.WorkspaceSizes)
    for call in CALLS:
        p = _pages(call)
        assert kernels.dll.roost_amd_cache_pages_workspace(ctx, C.addressof(p), C.addressof(sizes)) == abi.OK
        assert sizes.device_bytes > 12 * 64
        if call != "free":
            assert _run(kernels, ctx, call, p) == SMALL
    p.pages = 0
    assert kernels.dll.roost_amd_cache_pages_workspace(ctx, C.addressof(p), C.addressof(sizes)) == NOT
    p = _pages("free")
    p.count = 0
    assert _run(kernels, ctx, "free", p) == abi.OK


# ---- the definitions themselves ----------------------------------------------------------------------------------------------

def test_definition_of_the_format():
    """Every code stands for itself, and every value is off by at most one scale, half the grid's last step."""
    grid = torch.tensor(fc.GRID + [-g for g in fc.GRID])
    x = torch.zeros(1, 32)
    x[0, :16] = grid * 0.25
    codes, byte = fc.to_f4(x)
    assert codes[0, :16].tolist() == list(range(16)) and byte.tolist() == [[125]]
    g = torch.Generator().manual_seed(1)
    x = torch.randn(500, 64, generator=g) * torch.exp(5 * torch.randn(500, 1, generator=g))
    codes, byte = fc.to_f4(x)
    scale = torch.exp2(byte.double() - 127).repeat_interleave(32, 1)
    y = torch.tensor(fc.GRID + [-g for g in fc.GRID], dtype=torch.float64)[codes.long()] * scale
    assert ((x.double() - y).abs() <= scale).all()
    top = x.double().abs().reshape(500, 2, 32).amax(2)
    assert (top <= 7 * torch.exp2(byte.double() - 127)).all() and (top > 3.5 * torch.exp2(byte.double() - 127)).all()


def test_definition_of_the_pages():
    """A life of a small pool by the definitions: every page is held as often as refs says, at each step."""
    st = fc.Pages([[-1] * 4 for _ in range(6)], [0] * 6, [0] * 10, 16)

    def sound():
        held = [p for s in range(6) for p in st.held(s)]
        assert [held.count(p) for p in range(10)] == st.refs

    assert st.grow([0, 1], [0, 20, 50]) == ([1, 1], list(range(20)) + list(range(32, 62)))
    sound()
    assert st.fork([(0, 2), (1, 3), (0, 2)]) == ([1, 1, 0], [(1, 4), (3, 5)])
    sound()
    st.free([0])
    sound()
    assert st.tables[2][:2] == [0, 4] and st.refs == [1, 0, 2, 1, 1, 1, 0, 0, 0, 0]
    assert st.compact() == (5, [(5, 1)])
    sound()
    assert st.grow([2, 4], [0, 13, 14]) == ([1, 1], [4 * 16 + i for i in range(4, 16)] + [5 * 16] + [6 * 16])
    sound()
