"""CacheWriteF4 and CacheReadF4 on the GPU through the C ABI: codes, scales and values bit for bit against the definition."""
import math

import pytest
import torch

import f4_cases as fc
import roost_amd

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _check(session, k, v, slots, pages, heads, page, dim):
    """Writes k and v, compares the whole cache, reads the rows back."""
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = fc.random_cache(g, pages, heads, page, dim)
    want = [t.clone() for t in cache]
    named = torch.tensor(slots, dtype=torch.int64, device="cuda")
    live = [i for i, s in enumerate(slots) if 0 <= s < pages * page]
    at = torch.tensor([slots[i] for i in live], dtype=torch.long, device="cuda")
    for x, codes, scales in ((k, want[0], want[1]), (v, want[2], want[3])):
        if live:
            c, b = fc.to_f4(x[live].double())
            codes[at // page, :, at % page] = c[..., ::2] | c[..., 1::2] << 4
            scales[at // page, :, :, at % page] = b
    roost_amd.cache_write_f4(session, roost_amd.cache_f4_params(k, v, cache, named))
    for name, got, w in zip(roost_amd.CacheF4._fields, cache, want):
        assert torch.equal(got, w), name
    for back in (BF16, F32):
        out = [torch.full(k.shape, 7.0, dtype=back, device="cuda") for _ in range(2)]
        roost_amd.cache_read_f4(session, roost_amd.cache_f4_params(*out, cache, named))
        for got, codes, scales in ((out[0], *want[:2]), (out[1], *want[2:])):
            rows = fc.values(codes, scales)[at // page, :, at % page]
            assert torch.equal(torch.nan_to_num(got[live].double(), nan=-5.0), torch.nan_to_num(rows, nan=-5.0))
            dead = [i for i in range(len(slots)) if i not in set(live)]
            assert (got[dead] == 7).all()


def _rows(seed, tokens, heads, dim, dtype, gap=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((tokens, 2, heads * dim + gap), generator=g, device="cuda")
    x = x * torch.exp(3 * torch.randn((tokens, 2, 1), generator=g, device="cuda"))
    x = x.to(dtype)[:, :, :heads * dim].unflatten(2, (heads, dim))
    return x[:, 0], x[:, 1]


@pytest.mark.parametrize("tokens,heads,dim,page,dtype,gap", [
    (1, 2, 256, 16, BF16, 0), (1, 1, 64, 16, F32, 0), (7, 3, 64, 32, BF16, 8), (33, 8, 128, 64, F16, 0), (129, 5, 128, 16, F32, 16),
    (300, 2, 256, 128, BF16, 0), (1001, 8, 64, 1024, F16, 24)])
def test_write_and_read(session, tokens, heads, dim, page, dtype, gap):
    k, v = _rows(tokens, tokens, heads, dim, dtype, gap)
    pages = -(-2 * tokens // page)
    order = torch.randperm(pages * page, generator=torch.Generator().manual_seed(tokens)).tolist()
    slots = order[:tokens]
    slots[::5] = [(-1, -2 ** 40, pages * page, 2 ** 62, -2 ** 63)[i % 5] for i in range(len(slots[::5]))] if tokens > 1 else slots
    _check(session, k, v, slots, pages, heads, page, dim)


def test_contiguous_rows(session):
    k, v = (x.contiguous() for x in _rows(3, 40, 4, 128, BF16))
    _check(session, k, v, list(range(40)), 3, 4, 16, 128)


def test_every_rounding(session):
    """Each border between two codes, its neighbours on both sides, each block's largest value at and around 7 scales, ends of
    the range, zeros of both signs, infinities and NaN, one at a time in a block."""
    middles = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    cells = []
    for scale in (2.0 ** -120, 2.0 ** -119, 2.0 ** -3, 1.0, 2.0 ** 60, 2.0 ** 124, 2.0 ** 125):
        for m in middles + fc.GRID:
            for step in (-1, 0, 1):
                x = torch.tensor(m, dtype=F32)
                x = torch.nextafter(x, torch.tensor(math.inf * step)) if step else x
                cells.append([float(x) * scale, -float(x) * scale, 6 * scale])
        for top in (6.5, 6.9999995, 7.0, 7.0000005, 7.5):
            cells.append([min(top * scale, 3.4e38), -0.0, scale])
    for odd in (math.inf, -math.inf, math.nan, 3.4028234663852886e38, 1e-45, 2.0 ** -126, 2.0 ** -121, 0.0, -0.0):
        cells.append([odd, 1.0 if abs(odd) > 1e-30 or odd != odd else 0.0, -0.0])
    x = torch.zeros((len(cells), 1, 64), dtype=F32)
    for i, c in enumerate(cells):
        x[i, 0, 3:6] = torch.tensor(c, dtype=F32)
        x[i, 0, 32:] = torch.arange(32) * 0.25  # the block beside it is its own
    x = x.cuda()
    for dtype in (F32, BF16):
        y = x.to(dtype)
        _check(session, y, y.flip(0).contiguous(), list(range(len(cells))), -(-len(cells) // 16), 1, 16, 64)


def test_graph_and_stream(session):
    """Captured on a stream of its own and replayed over new rows and slots, beside eager work."""
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    k, v = (x.contiguous() for x in _rows(1, 50, 2, 128, BF16))
    slots = torch.arange(50, dtype=torch.int64, device="cuda")
    cache = roost_amd.cache_f4(5, 2, 16, 128)
    back = [torch.zeros_like(k), torch.zeros_like(v)]
    write = roost_amd.cache_f4_params(k, v, cache, slots)
    read = roost_amd.cache_f4_params(*back, cache, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.cache_write_f4(own, write)
        roost_amd.cache_read_f4(own, read)
    for i in range(4):
        a, b = _rows(10 + i, 50, 2, 128, BF16)
        k.copy_(a), v.copy_(b)
        slots.copy_(torch.randperm(80, device="cuda")[:50])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in ((k, back[0]), (v, back[1])):
            c, s = fc.to_f4(x.double())
            grid = torch.tensor(fc.GRID + [-t for t in fc.GRID], dtype=torch.float64, device="cuda")
            assert torch.equal(y.double(), grid[c.long()] * torch.exp2(s.double() - 127).repeat_interleave(32, -1))
    own.close()


def test_slots_past_4_gib(session):
    """Offsets that pass 32 bits: the last page of a pool of 4.4 GB of codes."""
    pages, heads, page, dim = 4200, 8, 1024, 256
    cache = roost_amd.cache_f4(pages, heads, page, dim)
    k, v = (x.contiguous() for x in _rows(9, 3, heads, dim, BF16))
    slots = [pages * page - 1, (pages - 1) * page + 5, 17]
    named = torch.tensor(slots, dtype=torch.int64, device="cuda")
    roost_amd.cache_write_f4(session, roost_amd.cache_f4_params(k, v, cache, named))
    for x, codes, scales in ((k, *cache[:2]), (v, *cache[2:])):
        c, b = fc.to_f4(x.double())
        for i, s in enumerate(slots):
            assert torch.equal(codes[s // page, :, s % page], c[i][..., ::2] | c[i][..., 1::2] << 4)
            assert torch.equal(scales[s // page, :, :, s % page], b[i])
        assert int(codes.sum(dtype=torch.int64)) == int(sum((c[i][..., ::2] | c[i][..., 1::2] << 4).long().sum() for i in range(3)))
