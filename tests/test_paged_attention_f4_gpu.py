"""PagedAttentionF4 on the GPU through the C ABI, against its definition in 64 bits; the bound is derived in f4_cases.py."""
import pytest
import torch

import f4_cases as fc
import roost_amd

pytestmark = pytest.mark.gpu

DECODE = [
    # lengths, query heads, KV heads, head dim, page
    ([(1, 1)], 8, 2, 256, 16),
    ([(1, 15), (1, 16), (1, 17), (1, 33)], 8, 2, 128, 16),
    ([(1, 1500)], 8, 2, 256, 16),
    ([(1, 700), (1, 1), (1, 1200), (1, 4097)], 32, 8, 128, 64),
    ([(1, 260), (1, 64)], 8, 8, 64, 16),      # one query head to each KV head
    ([(1, 500), (1, 31)], 6, 2, 64, 32),      # three
    ([(1, 500), (1, 129)], 16, 1, 128, 128),  # sixteen, one KV head
    ([(1, 300), (1, 77)], 32, 1, 256, 16),    # thirty-two: two tiles of rows
    ([(1, 300), (1, 1000)], 20, 1, 64, 1024),
    ([(2, 40), (3, 3), (1, 90), (4, 1000)], 8, 2, 128, 16),  # a few tokens each, as drafts have
    ([(5, 600), (7, 7)], 8, 2, 256, 16),      # more rows than a tile
]


@pytest.mark.parametrize("lens,q_heads,kv_heads,dim,page", DECODE)
@pytest.mark.parametrize("csr", [False, True])
def test_rows(session, lens, q_heads, kv_heads, dim, page, csr):
    a = fc.Attention(len(lens) + dim, lens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, csr=csr, pad=3)
    a.run(session)
    a.check()


PREFILL = [
    ([(17, 17)], 8, 2, 256, 16),
    ([(64, 64), (65, 190)], 8, 2, 128, 16),
    ([(300, 300)], 32, 8, 128, 64),
    ([(129, 1000), (1, 513), (33, 33)], 8, 2, 256, 16),
    ([(200, 1111), (1, 1), (1, 2000), (77, 78)], 16, 4, 64, 32),
    ([(511, 513)], 3, 1, 128, 16),
    ([(70, 400)], 32, 1, 64, 128),
    ([(90, 300), (2, 50)], 7, 1, 256, 1024),
    ([(1000, 1000)], 1, 1, 64, 16),
]


@pytest.mark.parametrize("lens,q_heads,kv_heads,dim,page", PREFILL)
@pytest.mark.parametrize("csr", [False, True])
def test_chunks(session, lens, q_heads, kv_heads, dim, page, csr):
    a = fc.Attention(len(lens) + dim, lens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, csr=csr, pad=2)
    a.run(session)
    a.check()


MIXED = [(1, 700), (130, 400), (1, 5), (3, 90), (40, 40)]


@pytest.mark.parametrize("kw", [
    dict(window=0), dict(window=1), dict(window=15), dict(window=16), dict(window=127), dict(window=5000), dict(soft_cap=30.0),
    dict(soft_cap=2.0, window=40), dict(causal=False), dict(scale=0.3), dict(slots=True), dict(gap=64), dict(hints=False),
    dict(hints=False, csr=True)], ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_options(session, kw, dim):
    a = fc.Attention(7, MIXED, dim=dim, page=32, **kw)
    a.run(session)
    a.check(str(kw))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("csr", [False, True])
def test_empty_rows(session, dim, csr):
    """Sequences without keys, without tokens, with more tokens than keys: rows that see nothing give 0 and minus infinity."""
    a = fc.Attention(11, [(1, 0), (0, 50), (6, 4), (1, 30), (50, 20), (0, 0), (2, 0)], dim=dim, csr=csr, pad=4)
    a.run(session)
    a.check()


def test_more_tokens_than_expected(session):
    """max_q_len and max_kv_len only say how the work is cut."""
    for hints in (dict(max_q_len=1, max_kv_len=16), dict(max_q_len=1, max_kv_len=100000), dict(max_q_len=9999, max_kv_len=1)):
        a = fc.Attention(12, [(1, 3000), (40, 700), (9, 9), (1, 100)], dim=128)
        a.hints = hints
        a.run(session)
        a.check(str(hints))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_bad_pages(session, dim):
    """Page ids outside the pool hold no keys, whichever place of a tile they have."""
    a = fc.Attention(13, [(1, 300), (100, 500), (3, 70)], dim=dim, page=16)
    for b, p in ((0, 0), (0, 7), (0, 18), (1, 3), (1, 4), (1, 31), (2, 4)):
        a.page_ids[b][p] = (-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1)[(b + p) % 4]
        a.table[b, p] = a.page_ids[b][p]
    a.run(session)
    a.check()


@pytest.mark.parametrize("csr", [False, True])
def test_tables_out_of_range(session, csr):
    """Rows of no table, lengths past the row, negative ones: no keys, or those that the row holds."""
    a = fc.Attention(14, [(1, 64), (2, 64), (1, 64), (20, 64)], dim=128, csr=csr, slots=not csr)
    if csr:
        a.indptr[-1] = 10 ** 9                 # past the entries: those that there are
        a.last[1] = 10 ** 6                    # more than a page
        a.last[0] = -5                         # less than nothing: the pages before it
        a.lens[0] = (1, 48)
        a.page_ids[0] = a.page_ids[0][:3]
    else:
        a.sequences[0], a.sequences[2] = -1, 10 ** 6
        a.keys[a.rows[1]], a.keys[a.rows[3]] = -7, 10 ** 9
        width = a.table.shape[1]
        a.lens = [(1, 0), (2, 0), (1, 0), (20, width * 16)]
        a.page_ids = [[], [], [], a.page_ids[3] + [-1] * (width - 4)]
    a.run(session)
    a.check()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("where", ["k", "v"])
def test_nan_blocks_stay_with_their_rows(session, dim, where):
    """A block of NaN reaches the rows that see its key (through v: in its dims alone) and no other: rows before it, other
    heads, other sequences, rows whose window has passed it, and nothing behind a sequence's last key."""
    for window in (-1, 20):
        a = fc.Attention(15, [(60, 200), (1, 100), (5, 90), (1, 333)], dim=dim, window=window)
        scales = a.cache[1 if where == "k" else 3]
        for b, key in ((0, 170), (0, 199), (2, 87), (3, 0), (3, 320)):
            scales[a.page_ids[b][key // 16], key % 2, key % (dim // 32), key % 16] = 255
        for b in range(4):  # behind the last key
            keys = a.lens[b][1]
            if keys % 16:
                for t in (a.cache[1], a.cache[3]):
                    t[a.page_ids[b][-1], :, :, keys % 16:] = 255
        a.run(session)
        a.check(f"window {window}")


def test_nan_queries(session):
    a = fc.Attention(16, [(40, 80), (1, 50)], dim=128)
    a.q[3, 1, 5] = float("nan")
    a.q[40, 2, 9] = float("nan")
    a.run(session)
    for token, head in ((3, 1), (40, 2)):
        assert torch.isnan(a.out[token, head]).all() and torch.isnan(a.lse[token, head])
        a.out[token, head], a.lse[token, head] = 0, 0
    assert torch.isfinite(a.out).all() and torch.isfinite(a.lse).all()


def test_large_scores(session):
    """Scores of thousands: one key takes all, the running maximum moves often."""
    a = fc.Attention(17, [(70, 600), (1, 900)], dim=128, std=60.0)
    a.run(session)
    a.check()


def test_many_sequences(session):
    g = torch.Generator().manual_seed(1)
    n = torch.randint(0, 4, (300,), generator=g).tolist()
    keys = torch.randint(0, 200, (300,), generator=g).tolist()
    n[17], n[230] = 90, 33
    lens = [(a, max(a, k)) for a, k in zip(n, keys)]
    a = fc.Attention(18, lens, q_heads=4, kv_heads=1, dim=64, pad=5)
    a.run(session)
    a.check()


def test_long_context(session):
    a = fc.Attention(19, [(1, 131072), (1, 70001)], q_heads=8, kv_heads=2, dim=128, page=64)
    a.run(session)
    a.check()
    a = fc.Attention(20, [(20, 40000)], q_heads=8, kv_heads=1, dim=256, page=64)
    a.run(session)
    a.check()


def test_offsets_past_4_gib(session):
    """A sequence whose pages lie beyond 4 GiB of codes."""
    heads, page, dim, pages = 8, 1024, 256, 4200
    a = fc.Attention(21, [(1, 3000), (30, 2050)], q_heads=8, kv_heads=8, dim=dim, page=page)
    big = roost_amd.cache_f4(pages, heads, page, dim)
    held = a.cache[0].shape[0]
    for t, s in zip(big, a.cache):
        t[pages - held:] = s
    a.table += torch.where(a.table >= 0, pages - held, 0).int()
    small, a.cache = a.cache, big
    a.run(session)
    a.cache = small  # the definition on the same pages under their old ids
    a.check()


def test_captured_once_serves_other_lengths(session):
    """One graph, replayed over other lengths, pages and queries, beside eager calls in a workspace of their own; every replay
    equals the eager call's bits."""
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    steps = [[(1, 100), (60, 300), (1, 7)], [(61, 200), (1, 1), (0, 0)], [(1, 900), (1, 40), (60, 64)], [(5, 640), (1, 3), (9, 1000)]]
    made = [fc.Attention(30 + i, lens, dim=128, spare=200) for i, lens in enumerate(steps)]
    a = made[0]
    width = 64
    cache = [torch.zeros((200, *t.shape[1:]), dtype=torch.uint8, device="cuda") for t in a.cache]
    q, out = torch.zeros((62, 8, 128), dtype=torch.bfloat16, device="cuda"), torch.empty((62, 8, 128), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((62, 8), device="cuda")
    cu, table, keys = fc.Attention.i32([0] * 4), fc.Attention.i32([[0] * width] * 3), fc.Attention.i32([0] * 3)
    make = lambda: roost_amd.paged_attention_f4_params(q, out, cache, cu, block_tables=table, kv_lens=keys, lse=lse)  # noqa: E731
    p = make()
    ws = roost_amd.paged_attention_f4_workspace(own, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.paged_attention_f4(own, p, ws)
    for _ in range(2):
        for m in made:
            n = m.q.shape[0]
            assert n <= 62
            q[:n] = m.q
            cu.copy_(m.cu)
            keys.copy_(m.keys)
            table.fill_(-1)
            table[:, :m.table.shape[1]] = m.table
            for t, s in zip(cache, m.cache):
                t[:min(200, s.shape[0])] = s[:200]
            out.fill_(7), lse.fill_(7)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone(), lse.clone()
            out.fill_(7), lse.fill_(7)
            roost_amd.paged_attention_f4(session, make())
            torch.cuda.synchronize()
            assert torch.equal(got[0].view(torch.int16), out.view(torch.int16)) and torch.equal(got[1], lse)
            if max(max(p) for p in m.page_ids if p) < 200:
                m.out, m.lse = got[0][:n], got[1][:n]
                m.check()
    own.close()


def test_same_bits_twice(session):
    a = fc.Attention(40, [(1, 5000), (300, 900), (1, 60)], dim=256)
    a.run(session)
    first = a.out.clone(), a.lse.clone()
    for _ in range(3):
        a.out.fill_(0)
        a.run(session)
        assert torch.equal(first[0], a.out) and torch.equal(first[1], a.lse)
