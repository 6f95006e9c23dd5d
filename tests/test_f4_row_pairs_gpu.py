"""PagedAttentionF4's row kernel with two tiles of 16 rows to a KV head: 17 to 32 rows at head_dim 64 and 128, which are a few draft
tokens of a group of query heads, or one token of a group above 16. Head_dim 256 takes the same rows in two turns and runs beside
them. Against the definition in 64 bits; the bound is derived in f4_cases.py."""
import random

import pytest
import torch

import f4_cases as fc
import roost_amd

pytestmark = pytest.mark.gpu

DIMS = [64, 128, 256]
SHAPES = [
    # lengths, query heads, KV heads, page
    ([(5, 700), (8, 9), (1, 33), (7, 2000)], 8, 2, 16),       # drafts: 5 to 8 tokens of 4 heads
    ([(3, 500), (4, 31), (4, 129), (2, 77)], 16, 2, 32),      # 3 and 4 of 8
    ([(17, 300), (32, 1000), (31, 31)], 3, 3, 64),            # 17 to 32 of one
    ([(9, 260), (10, 64), (1, 1)], 6, 2, 128),                # 9 and 10 of 3
    ([(2, 300), (2, 77)], 26, 2, 16),                         # 2 of 13
    ([(1, 1500), (1, 15), (1, 16), (1, 17)], 17, 1, 16),      # a token of 17 heads: one row in the second tile
    ([(1, 700), (1, 1), (1, 4097)], 48, 2, 64),               # of 24
    ([(1, 300), (1, 77), (1, 2000)], 96, 3, 1024),            # of 32
]


@pytest.mark.parametrize("lens,q_heads,kv_heads,page", SHAPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("csr", [False, True])
def test_rows(session, lens, q_heads, kv_heads, page, dim, csr):
    a = fc.Attention(len(lens) + dim, lens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page=page, csr=csr, pad=3)
    a.run(session)
    a.check()


# Drafts alone, and tokens of 20 heads beside prompt chunks.
MIXED = {"drafts": (dict(q_heads=8, kv_heads=2), [(8, 700), (5, 400), (1, 5), (3, 90), (7, 40), (8, 8)]),
         "groups": (dict(q_heads=40, kv_heads=2), [(1, 700), (130, 400), (1, 5), (3, 90), (1, 40), (1, 333)])}


def _mixed(seed, name, **kw):
    heads, lens = MIXED[name]
    return fc.Attention(seed, lens, **heads, **kw)


@pytest.mark.parametrize("kw", [
    dict(window=0), dict(window=1), dict(window=15), dict(window=16), dict(window=127), dict(window=5000), dict(soft_cap=30.0),
    dict(soft_cap=2.0, window=40), dict(causal=False), dict(causal=False, soft_cap=30.0), dict(scale=0.3), dict(slots=True),
    dict(gap=64), dict(hints=False), dict(hints=False, csr=True), dict(hints=False, soft_cap=30.0)], ids=str)
@pytest.mark.parametrize("name", MIXED)
@pytest.mark.parametrize("dim", DIMS)
def test_options(session, name, kw, dim):
    a = _mixed(7, name, dim=dim, page=32, **kw)
    a.run(session)
    a.check(str(kw))


EMPTY = {"drafts": (dict(q_heads=8, kv_heads=2), [(8, 0), (0, 50), (6, 4), (7, 30), (8, 5), (0, 0), (2, 0)]),
         "groups": (dict(q_heads=25, kv_heads=1), [(1, 0), (0, 50), (1, 30), (0, 0), (1, 4)])}


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("name", EMPTY)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("csr", [False, True])
def test_empty_rows(session, name, dim, csr, cap):
    """Rows that see no key, sequences without keys or tokens, rows of no sequence."""
    heads, lens = EMPTY[name]
    a = fc.Attention(11, lens, dim=dim, csr=csr, pad=4, soft_cap=cap, **heads)
    a.run(session)
    a.check()


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("name", MIXED)
@pytest.mark.parametrize("dim", DIMS)
def test_bad_pages(session, name, dim, cap):
    a = _mixed(13, name, dim=dim, page=16, soft_cap=cap)
    for b, p in ((0, 0), (0, 7), (0, 18), (0, 43), (1, 3), (1, 4), (1, 24), (3, 4)):
        a.page_ids[b][p] = (-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1)[(b + p) % 4]
        a.table[b, p] = a.page_ids[b][p]
    a.run(session)
    a.check()


@pytest.mark.parametrize("window", [-1, 20])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("name", MIXED)
@pytest.mark.parametrize("dim", DIMS)
def test_nan_blocks_stay_with_their_rows(session, name, dim, where, cap, window):
    """A block of NaN reaches the rows that see its key and no other, of either tile."""
    a = _mixed(15, name, dim=dim, window=window, soft_cap=cap)
    scales = a.cache[1 if where == "k" else 3]
    # Among the last tokens' own keys some rows see it and others do not; far before them all do, or none by the window.
    for b, key in ((0, 699), (0, 695), (0, 100), (1, 397), (3, 88), (5, a.lens[5][1] - 2), (5, 0)):
        scales[a.page_ids[b][key // 16], key % 2, key % (dim // 32), key % 16] = 255
    for b, (_, keys) in enumerate(a.lens):  # behind the last key
        if keys % 16:
            for t in (a.cache[1], a.cache[3]):
                t[a.page_ids[b][-1], :, :, keys % 16:] = 255
    a.run(session)
    a.check()


@pytest.mark.parametrize("dim", DIMS)
def test_nan_queries(session, dim):
    """One row of NaN in each tile, every other row as it would be."""
    a = fc.Attention(16, [(8, 80), (7, 500)], dim=dim)
    bad = ((0, 1), (7, 3), (8, 5), (14, 2))
    clean = a.q.clone()
    for token, head in bad:
        a.q[token, head, 5] = float("nan")
    a.run(session)
    for token, head in bad:
        assert torch.isnan(a.out[token, head]).all() and torch.isnan(a.lse[token, head])
    got = a.out.clone(), a.lse.clone()
    a.q.copy_(clean)
    a.run(session)
    for token, head in bad:
        for x, y in zip(got, (a.out, a.lse)):
            x[token, head] = y[token, head]
    assert torch.equal(got[0], a.out) and torch.equal(got[1], a.lse)
    a.check()


@pytest.mark.parametrize("dim", DIMS)
def test_large_scores(session, dim):
    """The running maximum moves often, in one tile and not in the other."""
    a = fc.Attention(17, [(8, 600), (5, 900)], dim=dim, std=60.0)
    a.run(session)
    a.check()


@pytest.mark.parametrize("dim", DIMS)
def test_more_tokens_than_expected(session, dim):
    """Hints of few rows: longer sequences take several turns of two tiles; hints of a draft, shorter ones leave rows empty."""
    for hints in (dict(max_q_len=8, max_kv_len=16), dict(max_q_len=5, max_kv_len=100000)):
        a = fc.Attention(12, [(1, 3000), (40, 700), (9, 9), (8, 100), (16, 2000)], dim=dim)
        a.hints = hints
        a.run(session)
        a.check(str(hints))


@pytest.mark.parametrize("dim", DIMS)
def test_long_context(session, dim):
    """Keys of one KV head over many workgroups, joined for rows of both tiles."""
    a = fc.Attention(19, [(8, 60001), (5, 9000)], q_heads=8, kv_heads=2, dim=dim, page=64)
    a.run(session)
    a.check()
    a = fc.Attention(20, [(1, 60001)], q_heads=32, kv_heads=1, dim=dim, page=64)
    a.run(session)
    a.check()


@pytest.mark.parametrize("batch", [64, 65, 704, 705])
@pytest.mark.parametrize("dim", [64, 128])
def test_batches(session, batch, dim):
    rng = random.Random(batch)
    lens = [(rng.choice([0, 1, 5, 8]), rng.randrange(200)) for _ in range(batch)]
    lens = [(min(n, k), k) for n, k in lens]
    lens[3] = (8, 3000)
    a = fc.Attention(batch, lens, q_heads=8, kv_heads=2, dim=dim, pad=1)
    a.run(session)
    a.check(some=set(rng.sample(range(batch), 40)) | {0, 3, batch - 1})


@pytest.mark.parametrize("dim", [64, 128])
def test_same_bits_twice_and_captured(session, dim):
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    a = fc.Attention(40, [(8, 5000), (5, 900), (7, 60)], dim=dim)
    a.run(session)
    torch.cuda.synchronize()
    first = a.out.clone(), a.lse.clone()
    p = a.params()
    ws = roost_amd.paged_attention_f4_workspace(own, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.paged_attention_f4(own, p, ws)
    for _ in range(3):
        a.out.fill_(0), a.lse.fill_(0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first[0], a.out) and torch.equal(first[1], a.lse)
        a.run(session)
        torch.cuda.synchronize()
        assert torch.equal(first[0], a.out) and torch.equal(first[1], a.lse)
    a.check()
    own.close()
