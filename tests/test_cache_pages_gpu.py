"""CacheCopy, CacheFork, CacheGrow, CacheFree and CacheCompact on the GPU through the C ABI, against host lists (f4_cases.Pages)
bit for bit."""
import random

import pytest
import torch

import f4_cases as fc
import roost_amd

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pools(seed, pages, shapes):
    """Pools [layers, pages, bytes]; a layer count below 0: layers further apart than their pages take."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for layers, size in shapes:
        gap = 3 if layers < 0 else 0
        t = torch.randint(0, 256, (abs(layers), pages + gap, size), dtype=torch.uint8, generator=g, device="cuda")
        out.append(t[:, :pages])
    return out


# ---- copies ----------------------------------------------------------------------------------------------------------------

COPIES = {
    "one": (10, [(3, 7)]),
    "apart": (40, [(i, 39 - i) for i in range(18)]),
    "onto itself": (5, [(2, 2), (1, 3)]),
    "chain": (12, [(0, 1), (1, 2), (2, 3), (5, 6)]),
    "backwards chain": (12, [(2, 3), (1, 2), (0, 1), (7, 8)]),
    "swap through a page": (12, [(0, 9), (1, 0), (9, 1)]),
    "one source for many": (30, [(4, i) for i in range(10, 30)]),
    "the same target": (30, [(i, 20) for i in range(9)] + [(21, 22)]),
    "the same pair twice": (30, [(1, 2), (1, 2), (2, 5)]),
    "outside": (8, [(0, 8), (-1, 2), (8, 3), (2 ** 31 - 1, 4), (5, -2 ** 31), (6, 7), (7, 1)]),
}


@pytest.mark.parametrize("name", COPIES)
@pytest.mark.parametrize("shapes", [[(1, 16)], [(3, 48), (2, 4096)], [(-2, 4112), (-3, 272), (1, 65536)]], ids=str)
def test_copies(session, name, shapes):
    pages, pairs = COPIES[name]
    pools = _pools(1, pages, shapes)
    want = [fc.copied(p, pairs) for p in pools]
    whole = [p._base.clone() if p._base is not None else None for p in pools]
    roost_amd.cache_copy(session, roost_amd.cache_copy_params(pools, _i32(pairs)))
    for p, w, before in zip(pools, want, whole):
        assert torch.equal(p, w)
        if before is not None:
            assert torch.equal(p._base[:, pages:], before[:, pages:])  # between the layers


@pytest.mark.parametrize("count", [255, 257, 1024, 1025, 5000])
@pytest.mark.parametrize("apart", [True, False])
def test_many_copies(session, count, apart):
    """Lists on both sides of the border between the two ways of telling which pairs meet."""
    rng = random.Random(count)
    pages = 3 * count
    pairs = [(rng.randrange(-1, pages + 1), rng.randrange(pages)) for _ in range(count)]
    if apart:
        order = rng.sample(range(pages), 2 * count)
        pairs = list(zip(order[::2], order[1::2]))
    pools = _pools(2, pages, [(2, 80), (1, 16)])
    want = [fc.copied(p, pairs) for p in pools]
    roost_amd.cache_copy(session, roost_amd.cache_copy_params(pools, _i32(pairs)))
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


def test_no_copies(session):
    pools = _pools(3, 4, [(1, 32)])
    before = pools[0].clone()
    roost_amd.cache_copy(session, roost_amd.cache_copy_params(pools, _i32([]).view(0, 2)))
    assert torch.equal(pools[0], before)


def test_copies_past_4_gib(session):
    pages, size = 40, 1 << 27
    pool = torch.zeros((1, pages, size), dtype=torch.uint8, device="cuda")
    pool[0, 39, :5] = torch.arange(1, 6, dtype=torch.uint8, device="cuda")
    pool[0, 39, -1] = 9
    roost_amd.cache_copy(session, roost_amd.cache_copy_params([pool], _i32([(39, 38), (38, 0)])))
    assert torch.equal(pool[0, 0], pool[0, 39]) and torch.equal(pool[0, 38], pool[0, 39]) and int(pool[0, 1].max()) == 0


# ---- tables ----------------------------------------------------------------------------------------------------------------

class State:
    """Tables on the GPU and on host lists, with pools."""

    def __init__(self, seed, *, sequences=12, live=7, width=9, pages=60, page=16, longest=None, shapes=((2, 64), (1, 4112))):
        rng = random.Random(seed)
        self.rng, self.page = rng, page
        tables = [[-1] * width for _ in range(sequences)]
        lengths, refs = [0] * sequences, [0] * pages
        order = rng.sample(range(pages), pages)
        for s in rng.sample(range(sequences), live):
            n = rng.randint(1, longest or width * page)
            k = -(-n // page)
            if len(order) < k:
                break
            tables[s][:k], order = order[:k], order[k:]
            lengths[s] = n
            for p in tables[s][:k]:
                refs[p] = 1
        self.host = fc.Pages([list(t) for t in tables], list(lengths), list(refs), page)
        self.tables, self.lengths, self.refs = _i32(tables), _i32(lengths), _i32(refs)
        self.pools = _pools(seed, pages, shapes)
        self.want = [p.clone() for p in self.pools]
        self.kw = dict(block_tables=self.tables, lengths=self.lengths, refs=self.refs, page_size=page)

    def live(self):
        return [s for s, n in enumerate(self.host.lengths) if n > 0]

    def empty(self):
        return [s for s, n in enumerate(self.host.lengths) if n == 0]

    def corrupt(self, s, b, page):
        self.tables[s, b] = page
        self.host.tables[s][b] = page

    def check(self, what):
        assert self.tables.tolist() == self.host.tables, what
        assert self.lengths.tolist() == self.host.lengths, what
        assert self.refs.tolist() == self.host.refs, what
        for got, want in zip(self.pools, self.want):
            assert torch.equal(got, want), what

    def fork(self, session, pairs):
        status = _i32([9] * len(pairs))
        roost_amd.cache_fork(session, roost_amd.cache_fork_params(self.pools, _i32(pairs).view(-1, 2), status, **self.kw))
        want, copies = self.host.fork(pairs)
        self.want = [fc.copied(p, copies) for p in self.want]
        assert status.tolist() == want
        self.check(f"fork {pairs}")
        return want

    def grow(self, session, requests, news):
        cu = [sum(news[:i]) for i in range(len(news) + 1)]
        slots = torch.full((cu[-1] + 3,), 77, dtype=torch.int64, device="cuda")
        status = _i32([9] * len(requests))
        roost_amd.cache_grow(session, roost_amd.cache_grow_params(_i32(requests), _i32(cu), slots, status, **self.kw))
        want, at = self.host.grow(requests, cu)
        assert status.tolist() == want and slots.tolist() == at + [77] * 3
        self.check(f"grow {requests} {news}")
        return want

    def free(self, session, requests):
        roost_amd.cache_free(session, roost_amd.cache_free_params(_i32(requests), **self.kw))
        self.host.free(requests)
        self.check(f"free {requests}")

    def compact(self, session):
        live = _i32([-1])
        roost_amd.cache_compact(session, roost_amd.cache_compact_params(self.pools, live, **self.kw))
        want, copies = self.host.compact()
        self.want = [fc.copied(p, copies) for p in self.want]
        assert live.tolist() == [want]
        self.check("compact")
        refs = self.refs.tolist()
        assert all(r > 0 for r in refs[:want]) and not any(r > 0 for r in refs[want:])


@pytest.mark.parametrize("page", [1, 16, 128])
def test_fork(session, page):
    st = State(1, page=page, width=9, pages=70)
    a, b = st.live()[:2]
    e = st.empty()
    st.fork(session, [(a, e[0]), (a, e[1]), (b, e[2])])
    st.fork(session, [(e[0], e[3]), (e[3], e[4])])  # a child's child; one whose parent this call makes is refused


def test_fork_refusals(session):
    st = State(2)
    a, b = st.live()[:2]
    e = st.empty()
    assert st.fork(session, [(a, b), (e[0], e[1]), (-1, e[1]), (99, e[1]), (a, -5), (a, 12), (a, a), (a, e[2]), (b, e[2]), (b, e[1])]) \
        == [0] * 7 + [1, 0, 0]  # the last one's child is named above


@pytest.mark.parametrize("left", [0, 1, 3])
def test_fork_without_pages(session, left):
    """Free pages run out: those that need none are served all the same."""
    st = State(3, sequences=20, live=6, page=16)
    whole, part = st.live()[:2]
    for s, n in ((whole, 32), (part, 33)):
        st.lengths[s] = n
        st.host.lengths[s] = n
    for p in [p for p, r in enumerate(st.host.refs) if r == 0][left:]:
        st.refs[p] = 5
        st.host.refs[p] = 5
    e = st.empty()
    got = st.fork(session, [(part, e[0]), (whole, e[1]), (part, e[2]), (part, e[3]), (whole, e[4]), (part, e[5])])
    assert got == [int(left > 0), 1, int(left > 1), int(left > 2), 1, 0]


def test_grow(session):
    st = State(4, pages=90)
    live, e = st.live(), st.empty()
    st.grow(session, [live[0], e[0], live[1], e[1], live[2]], [1, 17, 0, 16, 5])
    st.grow(session, [e[0], e[1]], [15, 1])


def test_grow_refusals(session):
    st = State(5, pages=40, width=6, longest=60)
    live, e = st.live(), st.empty()
    st.grow(session, [e[0], -1, 99, e[0], e[1], live[0]], [3, 4, 2, 5, 6 * 16 + 1, 1])
    # More pages than are left: this request and the later ones that need any.
    free = sum(r == 0 for r in st.host.refs)
    for p in [p for p, r in enumerate(st.host.refs) if r == 0][4:free]:
        st.refs[p] = 1
        st.host.refs[p] = 1
    assert st.grow(session, [e[1], e[2], e[3]], [40, 40, 1]) == [1, 0, 0]


def test_grow_many_tokens(session):
    st = State(6, sequences=5, live=2, width=700, pages=5000, page=16, longest=200, shapes=((1, 16),))
    e = st.empty()
    assert st.grow(session, [e[0], st.live()[0], e[1]], [11000, 999, 3]) == [1, 1, 1]


def test_short_slot_mapping(session):
    """Slots past the span are not written; the tables are as with all of them."""
    st = State(7)
    e = st.empty()[0]
    slots = torch.full((8,), 77, dtype=torch.int64, device="cuda")
    roost_amd.cache_grow(session, roost_amd.cache_grow_params(_i32([e, 99]), _i32([0, 20, 30]), slots[:5], None, **st.kw))
    _, at = st.host.grow([e, 99], [0, 20, 30])
    assert slots.tolist() == at[:5] + [77] * 3
    st.check("short")


def test_free(session):
    st = State(8)
    a, b, c = st.live()[:3]
    e = st.empty()
    st.fork(session, [(a, e[0]), (a, e[1])])
    st.free(session, [a, a, e[2], -3, 99, e[0]])
    st.free(session, [e[1], c])
    st.free(session, [])


def test_compact(session):
    st = State(9, pages=3000, sequences=60, live=40, width=30, shapes=((3, 64), (1, 1040)))
    st.compact(session)  # nothing below is free where nothing was freed; most seeds leave holes
    live = st.live()
    st.fork(session, [(live[0], st.empty()[0]), (live[1], st.empty()[1])])
    st.free(session, live[::2])
    st.compact(session)
    st.compact(session)  # nothing left to move
    st.free(session, st.live())
    st.compact(session)  # an empty pool


@pytest.mark.parametrize("pages", [1, 63, 64, 65, 1023, 1024, 1025, 2049])
def test_compact_sizes(session, pages):
    st = State(pages, pages=pages, sequences=8, live=6, width=max(1, pages // 7), page=16, shapes=((1, 16),))
    st.free(session, st.live()[:2])
    st.compact(session)
    st.free(session, st.live()[1:3])
    st.compact(session)


def test_full_pool(session):
    st = State(10, pages=64, sequences=4, live=4, width=16, page=16, shapes=((1, 16),))
    free = [p for p, r in enumerate(st.host.refs) if r == 0]
    for p in free:
        st.refs[p] = 1
        st.host.refs[p] = 1
    st.compact(session)


def test_entries_outside_the_pool(session):
    """Ids that name no page are left alone by every call."""
    st = State(11, sequences=14, live=5, pages=70)
    live, e = st.live(), st.empty()
    for s, b, p in ((live[0], 0, -1), (live[1], 1, 70), (live[2], 0, 2 ** 31 - 1), (live[3], 0, -2 ** 31)):
        st.corrupt(s, b, p)
    st.fork(session, [(live[0], e[0]), (live[1], e[1]), (live[2], e[2])])
    st.compact(session)
    st.free(session, live[:3])
    st.compact(session)


def test_many_requests(session):
    st = State(12, sequences=2000, live=900, width=3, pages=6000, page=16, shapes=((1, 16),))
    live, e = st.live(), st.empty()
    rng = random.Random(3)
    st.fork(session, [(rng.choice(live), c) for c in e[:1024]])
    rng.shuffle(e)
    st.grow(session, e[:1024], [rng.randint(0, 20) for _ in range(1024)])
    st.free(session, rng.sample(range(2000), 1024))
    st.compact(session)


def test_large_pool(session):
    """Four million pages: every chunk's count in one workgroup's LDS."""
    pages = 4 << 20
    st = State(13, sequences=4, live=3, width=9, pages=200, page=16, shapes=((1, 16),))
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[:200] = st.refs
    free = [pages - 1, pages - 1025, 3 << 20, 2 << 20]
    refs[free] = 0
    refs[:200] = torch.where(refs[:200] == 0, 1, refs[:200])
    e = st.empty()[0]
    kw = dict(st.kw, refs=refs)
    slots = torch.zeros(40, dtype=torch.int64, device="cuda")
    roost_amd.cache_grow(session, roost_amd.cache_grow_params(_i32([e]), _i32([0, 40]), slots, **kw))
    want = sorted(free)[:3]
    assert st.tables[e, :3].tolist() == want and slots.tolist() == [want[i // 16] * 16 + i % 16 for i in range(40)]
    pool = torch.zeros((1, pages, 16), dtype=torch.uint8, device="cuda")
    pool[0, -2] = 7
    live = _i32([0])
    refs[5] = 0
    roost_amd.cache_compact(session, roost_amd.cache_compact_params([pool], live, **kw))
    assert live.tolist() == [pages - 2] and bool((pool[0, 5] == 7).all())  # page 5 took the last used page, pages - 2
    used = refs.cpu()
    assert (used[:pages - 2] > 0).all() and (used[pages - 2:] == 0).all()


def test_captured(session):
    """One graph of free, fork, grow and compact, replayed over other tables beside eager work; two graphs share a workspace on
    one stream."""
    stream = torch.cuda.Stream()
    own = roost_amd.OpSession(session.lib, device=0, stream=stream)
    make = lambda seed: State(seed, sequences=20, live=9, width=6, pages=80, shapes=((2, 64), (1, 4112)))  # noqa: E731
    st = make(20)
    ended, pairs, grown = _i32([0] * 3), _i32([[0, 0]] * 3), _i32([0] * 3)
    cu, slots, live = _i32([0, 4, 5, 30]), torch.zeros(30, dtype=torch.int64, device="cuda"), _i32([0])
    calls = [(roost_amd.cache_free, roost_amd.cache_free_params(ended, **st.kw)),
             (roost_amd.cache_fork, roost_amd.cache_fork_params(st.pools, pairs, None, **st.kw)),
             (roost_amd.cache_grow, roost_amd.cache_grow_params(grown, cu, slots, None, **st.kw)),
             (roost_amd.cache_compact, roost_amd.cache_compact_params(st.pools, live, **st.kw))]
    roost_amd.cache_pages_workspace(own, calls[3][1])
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph, part in zip(graphs, (calls[:2], calls[2:])):
        with torch.cuda.graph(graph, stream=stream):
            for fn, p in part:
                fn(own, p)
    for seed in range(21, 26):
        new = make(seed)
        for a, b in zip((st.tables, st.lengths, st.refs, *st.pools), (new.tables, new.lengths, new.refs, *new.pools)):
            a.copy_(b)
        at, e = new.live(), new.empty()
        end, fork = at[:3], [(at[3], e[0]), (at[4], e[1]), (at[3], e[2])]
        grow = [e[0], at[5], e[3]]
        ended.copy_(_i32(end)), pairs.copy_(_i32(fork)), grown.copy_(_i32(grow))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay()
            graphs[1].replay()
        torch.cuda.synchronize()
        new.host.free(end)
        _, copies = new.host.fork(fork)
        _, at = new.host.grow(grow, [0, 4, 5, 30])
        count, moved = new.host.compact()
        assert slots.tolist() == at and live.tolist() == [count]
        assert st.tables.tolist() == new.host.tables and st.refs.tolist() == new.host.refs
        for got, pool in zip(st.pools, new.pools):
            assert torch.equal(got, fc.copied(pool, copies + moved))
    own.close()
