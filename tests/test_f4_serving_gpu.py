"""The 4-bit cache, its attention and the page calls together, as a server runs them: sequences grow, are written, answer, fork,
end, and the pool is made dense under those that stay. What every sequence should hold is kept on the side, token by token."""
import random

import pytest
import torch

import f4_cases as fc
import roost_amd

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


class Server:
    """Tables and `layers` caches on the GPU; the same tables as host lists; and each sequence's K and V rows as the cache has to
    hold them, [layer][K, V][tokens, kv_heads, dim] in 64 bits."""

    def __init__(self, session, *, layers=2, slots=7, pages=40, width=8, page=16, q_heads=8, kv_heads=2, dim=128, seed=0):
        self.session, self.layers, self.page, self.pages, self.width = session, layers, page, pages, width
        self.q_heads, self.kv_heads, self.dim = q_heads, kv_heads, dim
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        codes, scales = (layers, pages, kv_heads, page, dim // 2), (layers, pages, kv_heads, dim // 32, page)
        self.pools = [torch.zeros(s, dtype=torch.uint8, device="cuda") for s in (codes, scales, codes, scales)]
        self.tables = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(slots, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.kw = dict(block_tables=self.tables, lengths=self.lengths, refs=self.refs, page_size=page)
        self.host = fc.Pages([[-1] * width for _ in range(slots)], [0] * slots, [0] * pages, page)
        empty = torch.zeros((0, kv_heads, dim), dtype=torch.float64, device="cuda")
        self.rows = [[[empty, empty] for _ in range(layers)] for _ in range(slots)]

    def cache(self, layer):
        return roost_amd.CacheF4(*(p[layer] for p in self.pools))

    def new_rows(self, tokens):
        """A step's q, k and v of each layer as views of one projection."""
        width = (self.q_heads + 2 * self.kv_heads) * self.dim
        return torch.randn((self.layers, tokens, width), generator=self.g, device="cuda").to(BF16)

    def parts(self, qkv):
        q, k, v = qkv.split([n * self.dim for n in (self.q_heads, self.kv_heads, self.kv_heads)], -1)
        return q.unflatten(-1, (-1, self.dim)), k.unflatten(-1, (-1, self.dim)), v.unflatten(-1, (-1, self.dim))

    def buffers(self, tokens, batch):
        """What a step of up to `tokens` tokens of `batch` sequences reads and writes, at addresses that stay."""
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        return dict(qkv=self.new_rows(tokens), named=i32(batch), cu=i32(batch + 1), status=i32(batch),
                    slots=torch.zeros(tokens, dtype=torch.int64, device="cuda"),
                    out=torch.zeros((self.layers, tokens, self.q_heads, self.dim), dtype=BF16, device="cuda"),
                    lse=torch.zeros((self.layers, tokens, self.q_heads), device="cuda"))

    def calls(self, b, **hints):
        """The step's calls, in order."""
        out = [(roost_amd.cache_grow, roost_amd.cache_grow_params(b["named"], b["cu"], b["slots"], b["status"], **self.kw))]
        for layer in range(self.layers):
            q, k, v = self.parts(b["qkv"][layer])
            out.append((roost_amd.cache_write_f4, roost_amd.cache_f4_params(k, v, self.cache(layer), b["slots"])))
            out.append((roost_amd.paged_attention_f4, roost_amd.paged_attention_f4_params(
                q, b["out"][layer], self.cache(layer), b["cu"], block_tables=self.tables, kv_lens=self.lengths,
                sequences=b["named"], lse=b["lse"][layer], **hints)))
        return out

    def fill(self, b, news):
        """A step of news = {sequence: tokens}, in that order, into the buffers."""
        cu = [0]
        for n in news.values():
            cu.append(cu[-1] + n)
        named = list(news)
        b["cu"].copy_(torch.tensor(cu + [cu[-1]] * (b["named"].numel() - len(named)), dtype=torch.int32))
        b["named"].copy_(torch.tensor(named + [-1] * (b["named"].numel() - len(named)), dtype=torch.int32))
        b["qkv"].copy_(self.new_rows(b["qkv"].shape[1]))
        b["slots"].fill_(-1), b["status"].fill_(9), b["out"].fill_(7), b["lse"].fill_(7)

    def check_step(self, b, news, what):
        status, slots = self.host.grow(list(news), b["cu"].tolist()[:len(news) + 1])
        assert status == [1] * len(news), what
        assert b["status"].tolist()[:len(news)] == status and b["slots"].tolist()[:len(slots)] == slots, what
        at = 0
        for s, n in news.items():
            for layer in range(self.layers):
                for side, t in enumerate(self.parts(b["qkv"][layer])[1:]):
                    codes, bytes_ = fc.to_f4(t[at:at + n])
                    grid = torch.tensor(fc.GRID + [-x for x in fc.GRID], dtype=torch.float64, device="cuda")
                    held = grid[codes.long()] * torch.exp2(bytes_.double() - 127).repeat_interleave(32, -1)
                    self.rows[s][layer][side] = torch.cat([self.rows[s][layer][side], held])
            at += n
        self.check(what)
        for layer in range(self.layers):
            a = fc.Attention.__new__(fc.Attention)
            a.lens = [(n, self.host.lengths[s]) for s, n in news.items()]
            a.page_ids = [self.host.tables[s][:self.host.used(s)] for s in news]
            a.cache, a.q, a.out, a.lse = self.cache(layer), self.parts(b["qkv"][layer])[0], b["out"][layer], b["lse"][layer]
            a.q_heads, a.kv_heads, a.dim, a.page = self.q_heads, self.kv_heads, self.dim, self.page
            a.scale, a.window, a.soft_cap, a.causal = 0.0, -1, 0.0, True
            a.check(f"{what} layer {layer}")

    def check(self, what):
        """The tables, and what the pages that they name hold."""
        assert self.tables.tolist() == self.host.tables and self.lengths.tolist() == self.host.lengths, what
        assert self.refs.tolist() == self.host.refs, what
        for layer in range(self.layers):
            k, ks, v, vs = self.cache(layer)
            for side, held in enumerate((fc.values(k, ks), fc.values(v, vs))):
                for s, n in enumerate(self.host.lengths):
                    ids = torch.tensor(self.host.tables[s][:self.host.used(s)], dtype=torch.long, device="cuda")
                    got = held[ids].transpose(1, 2).reshape(-1, self.kv_heads, self.dim)[:n]
                    assert torch.equal(got, self.rows[s][layer][side]), f"{what}: sequence {s} layer {layer}"

    def step(self, news, **hints):
        b = self.buffers(sum(news.values()) + 2, len(news))
        self.fill(b, news)
        for fn, p in self.calls(b, **hints):
            fn(self.session, p)
        torch.cuda.synchronize()
        self.check_step(b, news, f"step {news}")

    def fork(self, pairs):
        status = torch.full((len(pairs),), 9, dtype=torch.int32, device="cuda")
        named = torch.tensor(pairs, dtype=torch.int32, device="cuda")
        roost_amd.cache_fork(self.session, roost_amd.cache_fork_params(self.pools, named, status, **self.kw))
        want, _ = self.host.fork(pairs)
        assert status.tolist() == want == [1] * len(pairs)
        for parent, child in pairs:
            self.rows[child] = [list(x) for x in self.rows[parent]]
        self.check(f"fork {pairs}")

    def free(self, ended):
        roost_amd.cache_free(self.session, roost_amd.cache_free_params(torch.tensor(ended, dtype=torch.int32, device="cuda"),
                                                                       **self.kw))
        self.host.free(ended)
        for s in ended:
            self.rows[s] = [[t[:0] for t in x] for x in self.rows[s]]
        self.check(f"free {ended}")

    def compact(self):
        live = torch.full((1,), -1, dtype=torch.int32, device="cuda")
        roost_amd.cache_compact(self.session, roost_amd.cache_compact_params(self.pools, live, **self.kw))
        want, _ = self.host.compact()
        assert live.tolist() == [want]
        self.check("compact")


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 16)])
def test_a_server_step_by_step(session, dim, page):
    s = Server(session, dim=dim, page=page, seed=dim)
    s.step({0: 20, 1: 33, 2: 1})                        # prompts
    s.step({0: 1, 1: 1, 2: 1}, max_q_len=1)             # a token each
    s.fork([(0, 3), (1, 5), (0, 4)])                    # answers side by side
    s.step({4: 1, 0: 1, 3: 1, 5: 2, 2: 30})             # each goes its own way; a chunk beside them
    s.free([0, 2])
    s.step({1: 1, 3: 1, 4: 1, 5: 1}, max_q_len=1)
    s.compact()
    s.step({3: 1, 5: 1, 4: 1, 0: 40})                   # a new prompt takes the pages that came free
    s.free([1, 3, 4, 5])
    s.compact()
    s.step({0: 1})
    s.free([0])
    s.compact()


def test_a_captured_step_among_eager_calls(session):
    """One token a sequence, captured with its grow, writes and attention; forks, ends, prompts and compaction come between its
    replays as eager calls. A batch with fewer sequences names -1 behind them."""
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    s = Server(session, slots=9, pages=60, seed=5)
    b = s.buffers(4, 4)
    calls = s.calls(b, max_q_len=1)
    for fn, p in calls:  # workspaces before the capture; with no sequence named the calls leave all as it was
        if fn is roost_amd.cache_grow:
            roost_amd.cache_pages_workspace(own, p)
        elif fn is roost_amd.paged_attention_f4:
            roost_amd.paged_attention_f4_workspace(own, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for fn, p in calls:
            fn(own, p)
    rng = random.Random(3)
    s.step({0: 17, 1: 16, 2: 40})
    for turn in range(8):
        live = [i for i, n in enumerate(s.host.lengths) if n]
        empty = [i for i, n in enumerate(s.host.lengths) if not n]
        if turn % 3 == 1:
            s.fork([(rng.choice(live), empty[0]), (rng.choice(live), empty[1])])
        if turn % 3 == 2:
            s.free(rng.sample(live, 2))
            s.compact()
        if turn == 4:
            s.step({empty[-1]: 23})
        live = [i for i, n in enumerate(s.host.lengths) if n]
        news = {i: 1 for i in rng.sample(live, min(4, len(live)))}
        s.fill(b, news)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s.check_step(b, news, f"replay {turn}")
    own.close()


def test_two_graphs_in_one_workspace(session):
    """Two captured calls of different shapes share a workspace and are replayed in turn."""
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    made = [fc.Attention(50, [(1, 3000), (1, 70), (1, 1)], dim=128), fc.Attention(51, [(40, 900), (1, 2000)], dim=256)]
    params = [a.params() for a in made]
    sizes = [roost_amd.paged_attention_f4_workspace(own, p, key=i) for i, p in enumerate(params)]
    ws = max(sizes, key=lambda w: w.device_bytes)
    torch.cuda.synchronize()
    graphs = []
    for p in params:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            roost_amd.paged_attention_f4(own, p, ws)
    for turn in range(3):
        for a in made:
            a.out.fill_(7), a.lse.fill_(7)
            a.q.copy_(torch.randn(a.q.shape, generator=a.g, device="cuda"))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for i in (0, 1, 0):
                graphs[i].replay()
        torch.cuda.synchronize()
        for a in made:
            a.check(f"turn {turn}")
    own.close()


@pytest.mark.parametrize("batch,most", [(64, 400), (65, 400), (703, 60), (704, 300), (705, 300), (1500, 90)])
@pytest.mark.parametrize("dim", [128, 256])
def test_batches_about_the_sizes_that_are_dealt(session, batch, most, dim):
    rng = random.Random(batch)
    lens = [(rng.choice([0, 1, 1, 1, 2]), rng.randrange(most)) for _ in range(batch)]
    lens = [(min(n, k), k) for n, k in lens]
    a = fc.Attention(batch, lens, q_heads=4, kv_heads=2, dim=dim, pad=1)
    a.run(session)
    a.check(some=set(rng.sample(range(batch), 60)) | {0, batch - 1})


def test_on_another_stream(session):
    """A call follows its session's stream: what that stream has yet to write is read after it is written."""
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    a = fc.Attention(60, [(1, 2000), (50, 300)], dim=128)
    p = a.params()
    q = a.q.clone()
    a.q.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        big = torch.randn((4096, 4096), device="cuda")
        for _ in range(8):
            big = big @ big * 1e-3
        a.q.copy_(q)
    roost_amd.paged_attention_f4(own, p)
    stream.synchronize()
    a.check()
    own.close()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_short_sequence_that_the_hints_rule_out(session, dim):
    """Two sequences of which max_q_len leaves neither short; one is, and one has no tokens at all."""
    for lens in ([(1, 500), (100, 300)], [(0, 40), (90, 90)], [(3, 3), (61, 70), (64, 900)]):
        a = fc.Attention(70, lens, dim=dim, pad=2)
        a.hints = dict(max_q_len=40, max_kv_len=100)
        a.run(session)
        a.check(str(lens))


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(96, 48, 64), (72, 24, 128), (130, 130, 64), (40, 40, 256)])
def test_many_heads(session, q_heads, kv_heads, dim):
    a = fc.Attention(80, [(1, 300), (2, 17), (90, 140), (1, 1)], q_heads=q_heads, kv_heads=kv_heads, dim=dim)
    a.run(session)
    a.check()


def test_a_sequence_named_twice(session):
    """Two entries of a batch may ask the same sequence."""
    a = fc.Attention(81, [(1, 700), (4, 700), (60, 700)], dim=128)
    a.sequences = a.i32([1, 1, 1])
    a.page_ids = [a.page_ids[1]] * 3
    a.run(session)
    a.check()


def test_two_calls_at_once(session):
    """Two sessions, a stream and a workspace each, on the same cache; neither waits for the other."""
    made = []
    for i in range(2):
        stream = torch.cuda.Stream()
        a = fc.Attention(82, [(1, 9000), (64, 2000), (1, 40)], dim=128)
        if i:
            a.q.copy_(torch.randn(a.q.shape, generator=a.g, device="cuda"))
            a.cache = made[0][1].cache
        made.append((roost_amd.OpSession(session.lib, device=0, stream=stream), a, a.params()))
    for own, _, p in made:
        roost_amd.paged_attention_f4_workspace(own, p)
    torch.cuda.synchronize()
    for _ in range(4):
        for own, _, p in made:
            roost_amd.paged_attention_f4(own, p)
    torch.cuda.synchronize()
    for own, a, _ in made:
        a.check()
        own.close()
