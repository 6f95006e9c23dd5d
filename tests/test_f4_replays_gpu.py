"""One captured PagedAttentionF4 call over steps of other lengths: every replay against the definition in 64 bits, and against an
eager call bit for bit. The steps share one pool, so each finds all of its keys there."""
import pytest
import torch

import f4_cases as fc
import roost_amd

pytestmark = pytest.mark.gpu

POOL, TOKENS, WIDTH, PAGE = 140, 70, 128, 16
STEPS = {
    "chunks": [[(1, 100), (60, 300), (1, 7)], [(61, 200), (1, 1), (0, 0)], [(1, 900), (1, 40), (60, 64)], [(5, 640), (1, 3), (9, 1000)],
               [(64, 2000), (0, 17), (2, 33)], [(1, 1), (1, 1), (1, 2000)]],
    "rows": [[(1, 100), (1, 1700), (1, 7)], [(1, 200), (1, 1), (0, 0)], [(8, 900), (5, 40), (1, 64)], [(3, 3), (0, 90), (8, 2000)]]}


@pytest.mark.parametrize("steps,hints", [
    ("chunks", {}), ("chunks", dict(max_q_len=64, max_kv_len=2048)), ("chunks", dict(max_q_len=16, max_kv_len=512)),
    ("rows", dict(max_q_len=8, max_kv_len=2048)), ("rows", dict(max_q_len=1, max_kv_len=100))], ids=str)
@pytest.mark.parametrize("csr", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_replays(session, steps, hints, csr, dim):
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    steps = STEPS[steps]
    blocks = [sum(-(-k // PAGE) for _, k in lens) for lens in steps]
    made = [fc.Attention(30 + i, lens, dim=dim, spare=POOL - n) for i, (lens, n) in enumerate(zip(steps, blocks))]
    heads = made[0].q.shape[1]
    cache = [torch.zeros_like(t) for t in made[0].cache]
    q, out = (torch.zeros((TOKENS, heads, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lse = torch.zeros((TOKENS, heads), device="cuda")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, table, keys, indptr, ids, last = i32(4), i32(3, WIDTH), i32(3), i32(4), i32(POOL), i32(3)
    tables = dict(kv_indptr=indptr, kv_indices=ids, kv_last_page_len=last) if csr else dict(block_tables=table, kv_lens=keys)
    p = roost_amd.paged_attention_f4_params(q, out, cache, cu, lse=lse, **tables, **hints)
    ws = roost_amd.paged_attention_f4_workspace(own, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.paged_attention_f4(own, p, ws)
    for turn in range(2):
        for m in made:
            n = m.q.shape[0]
            q[:n] = m.q
            cu.copy_(m.cu), keys.copy_(m.keys), indptr.copy_(m.indptr), last.copy_(m.last)
            table.fill_(-1), ids.fill_(-1)
            table[:, :m.table.shape[1]] = m.table
            ids[:m.ids.numel()] = m.ids
            for t, s in zip(cache, m.cache):
                t.copy_(s)
            out.fill_(7), lse.fill_(7)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone(), lse.clone()
            assert (out[n:] == 7).all() and (lse[n:] == 7).all()
            m.out, m.lse = got[0][:n], got[1][:n]
            m.check(f"turn {turn} {m.lens}")
            out.fill_(7), lse.fill_(7)
            roost_amd.paged_attention_f4(session, p)
            torch.cuda.synchronize()
            assert torch.equal(got[0].view(torch.int16), out.view(torch.int16)) and torch.equal(got[1], lse)
    own.close()
