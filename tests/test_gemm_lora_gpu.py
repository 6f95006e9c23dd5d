"""GemmLora on the GPU through the C ABI, against its definition in 64 bits; the bounds are derived in fused_cases.py."""
import pytest
import torch

import fused_cases
import roost_amd
from fused_cases import BF16, F32, F8, Lora

pytestmark = pytest.mark.gpu


def _run(session, c, key=0, **kw):
    roost_amd.gemm_lora(session, c.params(**kw), key=key)
    torch.cuda.synchronize()


CASES = {
    "one token": dict(lens=[1], slots=[2], in_dim=1024, out_dim=6144),
    "one token, one output": dict(lens=[1], slots=[0], in_dim=16, out_dim=1, adapters=1, max_rank=8),
    "one token, no adapter": dict(lens=[1], slots=[-1], in_dim=256, out_dim=100),
    "no adapters at all": dict(lens=[5, 9], slots=[0, 0], in_dim=264, out_dim=77, adapters=0, max_rank=0),
    "ragged": dict(lens=[5, 0, 33, 1, 0, 18], slots=[1, 0, 3, -1, 2, 1], in_dim=520, out_dim=613, ranks=[16, 3, 0, 9]),
    "decode": dict(lens=[1] * 61, slots=[(7 * i) % 25 - 1 for i in range(61)], in_dim=1024, out_dim=640, adapters=24,
                   max_rank=32, ranks=[1 + (5 * i) % 32 for i in range(24)], pad=3),
    "decode, 300 rows": dict(lens=[1] * 300, slots=[i % 5 - 1 for i in range(300)], in_dim=256, out_dim=200),
    "one adapter for all": dict(lens=[1] * 70, slots=[1] * 70, in_dim=512, out_dim=96),
    "slots outside the pool": dict(lens=[3, 3, 3], slots=[99, -7, 2], in_dim=128, out_dim=64),
    "mixed step": dict(lens=[1] * 48 + [200, 131], slots=[i % 4 for i in range(50)], in_dim=2048, out_dim=1024, addend=BF16),
    "prompt": dict(lens=[777], slots=[3], in_dim=1024, out_dim=1027, max_rank=64, ranks=[64, 64, 64, 57]),
    "prompts": dict(lens=[500, 3, 421], slots=[0, 1, 2], in_dim=1088, out_dim=515, max_rank=128, out=F32),
    "f32": dict(lens=[1, 40, 7], slots=[1, 0, -1], in_dim=516, out_dim=333, x=F32, out=F32, ranks=[16, 5, 2, 1]),
    "f32, many rows": dict(lens=[150, 170], slots=[1, 0], in_dim=260, out_dim=300, x=F32, out=F32, addend=F32),
    "8 bits, one token": dict(lens=[1], slots=[1], in_dim=1024, out_dim=800, x=F8),
    "8 bits": dict(lens=[30, 1, 1, 60], slots=[1, -1, 2, 0], in_dim=528, out_dim=275, x=F8, ranks=[16, 4, 1, 0], pad=5),
    "8 bits, prompts": dict(lens=[300, 290], slots=[1, 2], in_dim=1040, out_dim=520, x=F8, addend=BF16),
    "adapters alone": dict(lens=[1, 90, 17], slots=[1, -1, 0], in_dim=640, out_dim=321, shared=False, addend=BF16, pad=2),
    "adapters alone, no addend": dict(lens=[4, 60], slots=[1, -1], in_dim=640, out_dim=88, shared=False),
    "adapters alone, 8 bits": dict(lens=[200, 55], slots=[3, 1], in_dim=640, out_dim=328, shared=False, addend=BF16, x=F8),
    "strided rows": dict(lens=[20, 21], slots=[0, 3], in_dim=384, out_dim=101, x_gap=40, y_gap=3, addend=BF16),
    "strided prompts": dict(lens=[280, 41], slots=[0, 3], in_dim=384, out_dim=258, x_gap=40, y_gap=6, addend=F32),
    "f32 addend, f32 output": dict(lens=[9, 200], slots=[0, 3], in_dim=384, out_dim=128, addend=F32, out=F32),
}


@pytest.mark.parametrize("name", CASES)
def test_gemm_lora(session, name):
    c = Lora(len(name), **CASES[name])
    _run(session, c)
    c.check(name)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 400])
@pytest.mark.parametrize("x", [BF16, F8])
def test_numbers_of_rows(session, tokens, x):
    """Around every tile and wavefront border, in sequences of 1 to 40 rows."""
    lens, left = [], tokens
    while left:
        lens.append(min(left, 1 + (7 * len(lens)) % 40))
        left -= lens[-1]
    c = Lora(tokens, lens, [i % 6 - 1 for i in range(len(lens))], in_dim=272, out_dim=136, adapters=5, x=x, pad=1)
    _run(session, c)
    c.check(f"{tokens} rows")


@pytest.mark.parametrize("out_dim", [1, 3, 4, 15, 16, 17, 63, 64, 65, 127, 129, 255, 257])
@pytest.mark.parametrize("lens", [[3, 4], [150, 130]])
def test_numbers_of_outputs(session, out_dim, lens):
    c = Lora(out_dim, lens, [0, 1], in_dim=200, out_dim=out_dim)
    _run(session, c)
    c.check(f"{out_dim} outputs")


@pytest.mark.parametrize("in_dim", [8, 24, 56, 64, 72, 120, 136, 1000])
@pytest.mark.parametrize("lens", [[3, 4], [150, 130]])
def test_inner_lengths(session, in_dim, lens):
    c = Lora(in_dim, lens, [0, 1], in_dim=in_dim, out_dim=70)
    _run(session, c)
    c.check(f"inner length {in_dim}")


@pytest.mark.parametrize("max_rank", [8, 24, 40, 64, 72, 120, 128])
@pytest.mark.parametrize("lens", [[3, 1, 4], [150, 31, 130]])
def test_ranks(session, max_rank, lens):
    c = Lora(max_rank, lens, [0, 1, 2], in_dim=192, out_dim=80, adapters=3, max_rank=max_rank,
             ranks=[max_rank, max_rank - 7, max_rank // 2 + 1])
    _run(session, c)
    c.check(f"pool rank {max_rank}")


@pytest.mark.parametrize("lens", [[1] * 20, [150, 31, 130]])
def test_one_adapter_never_reaches_another_sequence(session, lens):
    """A broken adapter (NaN, infinities) leaves every other sequence's rows as they are without it, bit for bit; so does
    what the pool holds past an adapter's rank."""
    slots = [i % 3 for i in range(len(lens))]
    c = Lora(5, lens, slots, in_dim=256, out_dim=144, adapters=3, ranks=[16, 11, 5])
    _run(session, c)
    clean = c.y.clone()
    for pool, at in ((c.lora_a, (1, slice(None))), (c.lora_b, (1, slice(None)))):
        kept = pool.clone()
        pool[at] = float("nan")
        pool[1, :3] = float("inf")
        _run(session, c)
        row = 0
        for n, s in zip(lens, slots):
            mine = c.y[row:row + n]
            assert torch.isnan(mine).all() if s == 1 else torch.equal(mine, clean[row:row + n])
            row += n
        pool.copy_(kept)
    c.lora_a[1, 11:] = float("nan")
    c.lora_a[2, 5:] = float("inf")
    c.lora_b[1, :, 11:] = float("nan")
    c.lora_b[2, :, 5:] = float("inf")
    _run(session, c)
    assert torch.equal(c.y, clean)


@pytest.mark.parametrize("lens", [[4] * 10, [130, 128]])
def test_rows_of_no_sequence_may_hold_anything(session, lens):
    c = Lora(6, lens, [i % 3 for i in range(len(lens))], in_dim=256, out_dim=144, adapters=3, pad=9)
    c.x[sum(lens):] = float("nan")
    _run(session, c)
    c.check("NaN behind the last sequence")


@pytest.mark.parametrize("lens,x", [([1] * 9, BF16), ([300], BF16), ([7, 3], F32), ([200, 90], F8)])
def test_in_place_addend(session, lens, x):
    out = F32 if x == F32 else BF16
    c = Lora(7, lens, [i % 3 for i in range(len(lens))], in_dim=256, out_dim=144, adapters=3, x=x, out=out, addend=out)
    _run(session, c)
    want = c.y.clone()
    c.y = c.addend
    _run(session, c)
    assert torch.equal(c.y, want)


@pytest.mark.parametrize("lens", [[1] * 40, [260, 300]])
def test_same_bits_every_time(session, lens):
    c = Lora(8, lens, [i % 3 for i in range(len(lens))], in_dim=2048, out_dim=272, adapters=3)
    _run(session, c)
    first = c.y.clone()
    for _ in range(3):
        c.y.copy_(c.before)
        _run(session, c)
        assert torch.equal(c.y, first)


def test_two_sessions_at_once(session):
    """Calls on two streams with a workspace each."""
    cases = [Lora(20 + i, [70, 1, 30], [0, 1, 2], in_dim=1024, out_dim=520) for i in range(2)]
    sessions = [roost_amd.OpSession(session.lib, device=0, stream=torch.cuda.Stream()) for _ in range(2)]
    params = [c.params() for c in cases]
    spaces = [roost_amd.gemm_lora_workspace(s, p) for s, p in zip(sessions, params)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, p, w in zip(sessions, params, spaces):
            roost_amd.gemm_lora(s, p, w)
    torch.cuda.synchronize()
    for i, c in enumerate(cases):
        c.check(f"stream {i}")
    for s in sessions:
        s.close()


@pytest.mark.parametrize("lens", [[1] * 30, [200, 140]])
def test_graph_replays(session, lens):
    """Captured once, replayed with other rows, lengths and adapters in the same buffers and eager calls in between."""
    c = Lora(30, lens, [i % 4 for i in range(len(lens))], in_dim=512, out_dim=260, pad=4)
    stream = torch.cuda.Stream()
    s = roost_amd.OpSession(session.lib, device=0, stream=stream)
    p = c.params()
    ws = roost_amd.gemm_lora_workspace(s, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.gemm_lora(s, p, ws)
    for k in range(4):
        other = Lora(40 + k, lens, [(i + k) % 5 - 1 for i in range(len(lens))], in_dim=512, out_dim=260, pad=4)
        if k == 2:  # a shorter last sequence, more rows behind it
            other.lens = lens[:-1] + [max(lens[-1] - 1, 0)]
            other.cu[-1] -= 1
        for name in ("x", "cu", "slots_d", "y"):
            getattr(c, name).copy_(getattr(other, name))
        c.lens, c.slots, c.before = other.lens, other.slots, c.y.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check(f"replay {k}")
        got = c.y.clone()
        c.y.copy_(c.before)
        _run(session, c)
        assert torch.equal(got, c.y)
    s.close()


def test_large_offsets(session):
    """A weight and a pool whose elements pass 2^31 bytes."""
    c = Lora(50, [2, 17], [130, 3], in_dim=16384, out_dim=70000, adapters=131, max_rank=8)
    assert c.weight.numel() * 2 > 1 << 31
    _run(session, c)
    c.check("long offsets")


TYPES = [(BF16, BF16), (BF16, F32), (F32, F32), (F8, BF16), (F8, F32)]


# Sequences that share one launch with their low-rank rows: up to 8 rows, up to 16 ranks over all sequences; and one row more.
@pytest.mark.parametrize("x,out", TYPES)
@pytest.mark.parametrize("lens,max_rank", [([1], 16), ([8], 16), ([9], 16), ([1], 8), ([3, 5], 8), ([0, 4], 8), ([2, 0], 8),
                                           ([1, 1], 8), ([1], 24), ([2, 2, 2], 8)])
def test_few_rows(session, lens, max_rank, x, out):
    for k, (in_dim, out_dim, pad) in enumerate([(1024, 613, 0), (48, 16, 2), (1040, 5, 1)]):
        pad = min(pad, max(0, 8 - sum(lens)))
        slots = [(k + 2 * i) % 5 - 1 for i in range(len(lens))]
        c = Lora(60 + k, lens, slots, in_dim=in_dim, out_dim=out_dim, adapters=4, max_rank=max_rank,
                 ranks=[max_rank, 3, 0, 1 + max_rank // 2], x=x, out=out, addend=[None, BF16, F32][k], pad=pad,
                 x_gap=[0, 16, 32][k], y_gap=[0, 1, 3][k])
        _run(session, c)
        c.check(f"{lens} rows, inner length {in_dim}")


@pytest.mark.parametrize("x", [BF16, F32, F8])
def test_few_rows_keep_apart(session, x):
    """Of two sequences in one launch: NaN in one's adapter, rows or past its rank does not reach the other's rows."""
    out = F32 if x == F32 else BF16
    c = Lora(70, [3, 2], [1, 2], in_dim=640, out_dim=77, adapters=3, max_rank=8, ranks=[8, 6, 5], x=x, out=out, pad=1)
    _run(session, c)
    clean = c.y.clone()
    c.lora_a[1, 6:] = c.lora_a[2, 5:] = c.lora_a[0] = float("nan")
    c.lora_b[1, :, 6:] = c.lora_b[2, :, 5:] = c.lora_b[0] = float("inf")
    _run(session, c)
    assert torch.equal(c.y, clean)
    c.lora_a[2, 0] = float("nan")
    c.lora_b[2, :, 1] = float("-inf")
    _run(session, c)
    assert torch.equal(c.y[:3], clean[:3]) and torch.isnan(c.y[3:5]).all()
    if x != F8:  # rows of NaN
        c.x[4] = float("nan")
        c.x[5] = float("nan")
        _run(session, c)
        assert torch.equal(c.y[:3], clean[:3]) and torch.equal(c.y[5:], clean[5:])


def test_few_rows_replayed(session):
    c = Lora(71, [1], [2], in_dim=1024, out_dim=640)
    stream = torch.cuda.Stream()
    s = roost_amd.OpSession(session.lib, device=0, stream=stream)
    p = c.params()
    ws = roost_amd.gemm_lora_workspace(s, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.gemm_lora(s, p, ws)
    for k in range(4):
        other = Lora(72 + k, [1], [k - 1], in_dim=1024, out_dim=640)
        for name in ("x", "slots_d", "y"):
            getattr(c, name).copy_(getattr(other, name))
        c.slots, c.before = other.slots, c.y.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check(f"replay {k}")
    s.close()


def _lens(tokens, long):
    """Sequences of one token to `long`, and empty ones."""
    lens, left, k = [], tokens, 0
    while left:
        lens.append(min(left, [1, long, 1, 0, 3, long // 2, 17, 1][k % 8]))
        left -= lens[-1]
        k += 1
    return lens


# Rows x outputs that take each of the tilings of many rows, with sequences that start and end inside the tiles.
@pytest.mark.parametrize("x,out", TYPES)
@pytest.mark.parametrize("tokens,out_dim,long", [
    (13, 5001, 5),      # 32 outputs x 16 rows
    (31, 5001, 9),      # 32 x 32
    (40, 20500, 9),     # 32 x 64, more than one round
    (300, 2100, 90),    # 80 x 64
    (130, 8300, 1),     # 80 x 64, a sequence a row
    (300, 5001, 90),    # 64 x 64
    (1020, 2100, 400),  # 128 x 128
    (1100, 2100, 2),    # 128 x 128, a sequence a row or two
    (1500, 2901, 300),  # 256 x 128
    (1500, 2900, 3),
    (2601, 4200, 900),  # 256 x 256
    (2600, 4203, 4),    # 256 x 256, short sequences
    (4201, 4200, 700),  # 256 x 256 for 3,840 rows, 128 x 128 for the rest
    (4200, 4203, 5),
    (5201, 4200, 900),  # 256 x 256 for 3,840 rows, 256 x 128 for the rest
])
def test_tilings(session, tokens, out_dim, long, x, out):
    lens = _lens(tokens, long)
    c = Lora(80, lens, [(5 * i) % 8 - 1 for i in range(len(lens))], in_dim=144, out_dim=out_dim, adapters=7, max_rank=40,
             ranks=[40, 1, 16, 33, 0, 24, 39], x=x, out=out, pad=7)
    _run(session, c)
    c.check(f"{tokens} x {out_dim}")


@pytest.mark.parametrize("x", [BF16, F32, F8])
@pytest.mark.parametrize("tokens,out_dim,long", [(300, 5001, 90), (2600, 1100, 4), (4000, 640, 1500)])
def test_tilings_of_adapters_alone(session, tokens, out_dim, long, x):
    lens = _lens(tokens, long)
    out = F32 if x == F32 else BF16
    c = Lora(81, lens, [(5 * i) % 8 - 1 for i in range(len(lens))], in_dim=144, out_dim=out_dim, adapters=7, max_rank=128,
             ranks=[128, 1, 16, 33, 0, 24, 97], x=x, out=out, shared=False, addend=out, pad=3)
    _run(session, c)
    c.check(f"{tokens} x {out_dim}")


@pytest.mark.parametrize("x,out", TYPES)
@pytest.mark.parametrize("max_rank", [16, 32, 128])
def test_low_rank_rows_of_long_prompts(session, max_rank, x, out):
    """Pieces of 64 rows of one sequence, from sequences that start and end anywhere."""
    lens = [3001, 1, 0, 62, 2900, 300]
    c = Lora(82, lens, [0, 1, 2, 3, 1, 2], in_dim=400, out_dim=72, max_rank=max_rank,
             ranks=[max_rank, max_rank - 1, 3, 9], x=x, out=out, pad=2)
    _run(session, c)
    c.check(f"pool rank {max_rank}")


@pytest.mark.parametrize("each", [1, 2])
def test_more_sequences_than_a_workgroup_has_threads(session, each):
    lens = [each] * 1300
    lens[5] = lens[700] = 0
    c = Lora(83, lens, [(3 * i) % 12 - 1 for i in range(1300)], in_dim=128, out_dim=96, adapters=11)
    _run(session, c)
    c.check(f"1300 sequences of {each}")


@pytest.mark.parametrize("tokens", [6, 30, 300])
def test_ranks_outside_the_pool(session, tokens):
    """Ranks below zero count as none, above the pool's as the pool's."""
    c = Lora(84, [tokens // 3] * 3, [0, 1, 2], in_dim=256, out_dim=100, adapters=3, ranks=[-5, 1 << 30, 7])
    _run(session, c)
    c.check("ranks")


@pytest.mark.parametrize("lens", [[1], [2] * 20, [1000]])
def test_two_graphs_that_share_a_workspace(session, lens):
    """Replayed one after the other on one stream."""
    cases = [Lora(85 + i, lens, [i + 1] * len(lens), in_dim=512, out_dim=260) for i in range(2)]
    stream = torch.cuda.Stream()
    s = roost_amd.OpSession(session.lib, device=0, stream=stream)
    params = [c.params() for c in cases]
    ws = roost_amd.gemm_lora_workspace(s, params[0])
    torch.cuda.synchronize()
    graphs = []
    for p in params:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            roost_amd.gemm_lora(s, p, ws)
    for _ in range(3):
        for c in cases:
            c.y.copy_(c.before)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        for c in cases:
            c.check("replayed")
    s.close()


def test_a_graph_keeps_its_workspace_when_the_session_needs_a_larger_one(session):
    c = Lora(90, [20, 30], [1, 2], in_dim=512, out_dim=260)
    big = Lora(91, [2000], [1], in_dim=512, out_dim=64)
    stream = torch.cuda.Stream()
    s = roost_amd.OpSession(session.lib, device=0, stream=stream)
    p, q = c.params(), big.params()
    first = roost_amd.gemm_lora_workspace(s, p).device
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.gemm_lora(s, p)
    roost_amd.gemm_lora(s, q)
    torch.cuda.synchronize()
    taken = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")  # what a freed workspace's memory would be given to
    assert roost_amd.gemm_lora_workspace(s, p).device != first
    assert not any(t.data_ptr() < first + 256 and first < t.data_ptr() + t.numel() for t in (taken, big.y, c.y))
    for _ in range(2):
        c.y.copy_(c.before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check("replayed beside a larger workspace")
    assert (taken == 0).all()
    big.check("the larger call")
    s.close()


def test_other_sessions_device_is_refused(session):
    c = Lora(92, [2], [1], in_dim=64, out_dim=16)
    p = c.params()
    p._device = torch.device("cuda", 1)
    with pytest.raises(ValueError, match="session on"):
        roost_amd.gemm_lora(session, p)


# Tiles of many rows with few and many adapters each, which come again and again among their rows.
@pytest.mark.parametrize("x,out", TYPES)
@pytest.mark.parametrize("max_rank,adapters", [(8, 3), (8, 70), (16, 5), (16, 41), (24, 9), (32, 30), (64, 6)])
@pytest.mark.parametrize("tokens,out_dim", [(100, 12200), (300, 5001), (1500, 2901)])
def test_adapters_of_a_tile(session, tokens, out_dim, max_rank, adapters, x, out):
    lens = _lens(tokens, 20)
    c = Lora(86, lens, [(11 * i + i // 7) % (adapters + 1) - 1 for i in range(len(lens))], in_dim=80, out_dim=out_dim,
             adapters=adapters, max_rank=max_rank,
             ranks=[(max_rank, 1, 5, 0, max_rank - 1, 8)[i % 6] for i in range(adapters)],
             x=x, out=out, pad=2)
    _run(session, c)
    c.check(f"{adapters} adapters of rank {max_rank}")


@pytest.mark.parametrize("max_rank", [8, 16, 32, 48])
def test_adapters_of_a_tile_keep_apart(session, max_rank):
    """Broken adapters among others in a tile, and what the pool holds past the others' ranks."""
    lens = [1, 2] * 110
    slots = [i % 7 for i in range(220)]
    c = Lora(87, lens, slots, in_dim=128, out_dim=6000, adapters=7, max_rank=max_rank,
             ranks=[max_rank, 3, max_rank - 1, 0, 7, 8, 1])
    _run(session, c)
    clean = c.y.clone()
    for a, r in enumerate(c.ranks_h):
        c.lora_a[a, r:] = float("nan")
        c.lora_b[a, :, r:] = float("inf")
    c.lora_a[2] = float("nan")
    c.lora_b[4] = float("inf")
    _run(session, c)
    rows = torch.tensor([s for n, s in zip(lens, slots) for _ in range(n)], device="cuda")
    hit = (rows == 2) | (rows == 4)
    assert torch.equal(c.y[~hit], clean[~hit]) and not torch.isfinite(c.y[hit]).any()


# Tables that the documentation rules out: past the call's rows, backwards, below zero. Each ends in what belongs to the call.
# 33 to 65 rows and 300 by 80 outputs: tiles whose last rows start past the call's; the others: the tiles of many rows.
@pytest.mark.parametrize("x,out", [(BF16, BF16), (F8, BF16), (F32, F32)])
@pytest.mark.parametrize("tokens,out_dim", [(6, 40), (15, 40), (31, 300), (33, 40), (40, 9000), (65, 40), (300, 2100), (300, 5001),
                                            (1020, 2100), (1500, 2901)])
def test_a_broken_table_writes_nothing_behind_the_call(session, tokens, out_dim, x, out):
    first = tokens // 3
    c = Lora(93, [first, tokens - first], [1, 2], in_dim=144, out_dim=out_dim, max_rank=8, x=x, out=out, addend=out)
    want, bound = c.want()
    guard = 300  # rows behind the call's, in the same allocations
    wide = {}
    for name in ("y", "addend", "x_scale"):
        t = getattr(c, name)
        if t is not None:
            wide[name] = torch.cat([t, torch.full((guard, *t.shape[1:]), 7.0, device="cuda").to(t.dtype)])
            setattr(c, name, wide[name][:tokens])
    big = (1 << 31) - 1
    for table in ([0, first, tokens + 200], [0, first, big], [0, tokens + 200, tokens], [0, big, tokens], [-big, first, big],
                  [0, first, -5], [tokens + 7, tokens + 9, big]):
        c.cu.copy_(torch.tensor(table, dtype=torch.int32))
        wide["y"][:tokens] = c.before
        _run(session, c)
        assert all((t[tokens:].float() == 7).all() for t in wide.values()), table
        if table[0] <= 0 and table[1] == first:  # the first sequence is as it should be
            fused_cases.assert_within(c.y[:first], want[:first], bound[:first], str(table))


# Rows and outputs on both sides of where 256 x 128 tiles would take a second round of the CUs and 256 x 256 tiles begin.
@pytest.mark.parametrize("x,out", [(BF16, BF16), (F8, BF16), (F32, F32)])
@pytest.mark.parametrize("tokens,out_dim", [(2048, 4096), (2049, 4096), (2303, 4090), (2049, 3700), (384, 21700), (385, 21700)])
def test_where_the_largest_tiles_begin(session, tokens, out_dim, x, out):
    lens = _lens(tokens, 500)
    c = Lora(94, lens, [(3 * i) % 5 - 1 for i in range(len(lens))], in_dim=208, out_dim=out_dim, ranks=[16, 5, 0, 9], x=x, out=out)
    _run(session, c)
    c.check(f"{tokens} x {out_dim}")
