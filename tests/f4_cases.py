"""The 4-bit cache, its attention and the page calls by their definitions, in plain Python and 64 bits, and the error bounds
that the tests hold the kernels to.

Writing and reading a cache and all page calls are exact: their tests compare bits.

Attention. Per query row, with u = 2^-23 for an f32 operation (2^-23, not 2^-24: nothing says that a matrix instruction rounds
its inner sums to nearest) and d = head_dim:
  * a score is a sum of d products, off by at most (d + 4) u scale sum_i |q_i k_i| (bf16 and 4-bit products are exact in f32; 4
    for the products with scale and log2(e)); a soft cap adds 8 u cap (its exponential and reciprocal, off by an ulp each, and
    two roundings, all of numbers up to 2 cap);
  * a score off by e makes its p off by at most 2 e of it (e < 1/2), the exponent's own f32 argument, off by |s| u, by 2 |s| u,
    v_exp_f32 by u: SCORE = 2 e + 2 |s| u + u, with the largest |s| of the row;
  * sums over `keys` terms: keys u of the sum of magnitudes;
  * p is rounded to bf16 once, 2^-8 of it, and the output once more, 2^-8 of it;
  * p counts from a maximum that is not above the row's own, so the row's largest is 1 or more and their sum too: what v_exp_f32
    takes for zero, below 2^-126, is less than 2^-126 of the sum. An output below 2^-126 is rounded to a multiple of 2^-133.
So |out - want| <= 2^-8 |want| + (1 + 2^-7) (2^-8 + 2 (SCORE + keys u)) sum_j p_j |v_j| (p's error counts twice: in the sum over
v and in the sum of p) + 2^-126 sum_j |v_j| + 2^-133, and |lse - want| <= (SCORE + keys u) log2(e) + 4 u |want|.
"""
import math

import torch

U = 2.0 ** -23
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---- the format ---------------------------------------------------------------------------------------------------------

def to_f4(x):
    """(codes 0..15, scale bytes) of rows [..., dim] by the definition, in 64 bits."""
    cells = x.double().reshape(*x.shape[:-1], -1, 32)
    top = cells.abs().amax(-1)
    finite = torch.isfinite(cells).all(-1)
    top = torch.where(finite, top, torch.ones_like(top))
    # The smallest power of two s with top <= 7 s.
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -200) / 7)) - 1
    for _ in range(3):
        e = torch.where(top > 7 * torch.exp2(e), e + 1, e)  # exp2 of a whole number is exact, pow is not
    e = e.clamp(-120, 125)
    r = cells.abs() / torch.exp2(e)[..., None]
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    middles = (grid[1:] + grid[:-1]) / 2
    code = (r[..., None] > middles).sum(-1)
    tie = (r[..., None] == middles).any(-1) & (code % 2 == 1)  # between an odd code and the even one above it
    code = torch.where(tie, code + 1, code)
    code = torch.where(finite[..., None], code + 8 * torch.signbit(cells), torch.zeros_like(code))
    byte = torch.where(finite, e + 127, torch.full_like(e, 255))
    return code.reshape(x.shape).to(torch.uint8), byte.to(torch.uint8)


def values(codes, scales):
    """[pages, heads, page, dim] in 64 bits of a cache's packed codes and scale bytes."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    grid = torch.tensor(GRID + [-g for g in GRID], dtype=torch.float64, device=codes.device)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales > 252, torch.full_like(s, math.nan), s)
    return grid[c] * s.transpose(-1, -2).repeat_interleave(32, -1)


def random_cache(g, pages, heads, page, dim, device="cuda"):
    """Any codes, scales about 2^-2."""
    r = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=device, dtype=torch.int32).to(torch.uint8)  # noqa: E731
    return tuple(r(lo, hi, pages, heads, *s) for lo, hi, s in ((0, 256, (page, dim // 2)), (123, 127, (dim // 32, page))) * 2)


# ---- attention -------------------------------------------------------------------------------------------------------------

class Attention:
    """One call's inputs: lens = [(new tokens, keys with them), ...]; pad: rows of no sequence behind them."""

    def __init__(self, seed, lens, *, q_heads=8, kv_heads=2, dim=128, page=16, pad=0, csr=False, window=-1, soft_cap=0.0,
                 causal=True, scale=0.0, slots=False, gap=0, std=1.0, hints=True, spare=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.lens, self.csr, self.window, self.soft_cap, self.causal = g, lens, csr, window, soft_cap, causal
        self.q_heads, self.kv_heads, self.dim, self.page, self.scale = q_heads, kv_heads, dim, page, scale
        blocks = [-(-k // page) for _, k in lens]
        pages = sum(blocks) + spare
        self.cache = random_cache(g, pages, kv_heads, page, dim)
        order = torch.randperm(pages, generator=g, device="cuda").tolist()
        self.page_ids, at = [], 0
        for b in blocks:
            self.page_ids.append(order[at:at + b])
            at += b
        tokens = sum(n for n, _ in lens) + pad
        wide = torch.randn((tokens, q_heads * dim + gap), generator=g, device="cuda") * std
        self.q = wide.to(torch.bfloat16)[:, :q_heads * dim].unflatten(1, (q_heads, dim))
        self.out = torch.full((tokens, q_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        self.lse = torch.full((tokens, q_heads), 7.0, device="cuda")
        self.cu = self.i32([sum(n for n, _ in lens[:i]) for i in range(len(lens) + 1)])
        width = max(blocks + [1]) + 1
        rows = [p + [-1] * (width - len(p)) for p in self.page_ids]
        self.rows = list(range(len(lens)))
        keys = [k for _, k in lens]
        if slots:  # the batch names its rows of a larger table, in another order
            self.rows = [2 * i + 1 for i in reversed(range(len(lens)))]
            table, held = [[-1] * width for _ in range(2 * len(lens) + 1)], [0] * (2 * len(lens) + 1)
            for r, p, k in zip(self.rows, rows, keys):
                table[r], held[r] = p, k
            rows, keys = table, held
        self.table, self.keys = self.i32(rows), self.i32(keys)
        self.sequences = self.i32(self.rows) if slots else None
        self.indptr = self.i32([sum(blocks[:i]) for i in range(len(blocks) + 1)])
        self.ids = self.i32([p for ps in self.page_ids for p in ps] or [0])
        self.last = self.i32([k - (b - 1) * page if b else 0 for (_, k), b in zip(lens, blocks)])
        self.hints = dict(max_q_len=max(n for n, _ in lens), max_kv_len=max(k for _, k in lens)) if hints else {}

    @staticmethod
    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def params(self, **kw):
        import roost_amd

        args = dict(kv_indptr=self.indptr, kv_indices=self.ids, kv_last_page_len=self.last) if self.csr else \
            dict(block_tables=self.table, kv_lens=self.keys, sequences=self.sequences)
        args.update(lse=self.lse, window_left=self.window, soft_cap=self.soft_cap, causal=self.causal, sm_scale=self.scale,
                    **self.hints)
        args.update(kw)
        return roost_amd.paged_attention_f4_params(self.q, self.out, self.cache, self.cu, **args)

    def run(self, session, **kw):
        import roost_amd

        roost_amd.paged_attention_f4(session, self.params(**kw))

    def check(self, what="", some=None):
        """Every row (or the sequences `some`) within the bound, and rows of no sequence as they were."""
        k_all, v_all = values(*self.cache[:2]), values(*self.cache[2:])
        group, at = self.q_heads // self.kv_heads, 0
        scale = self.scale or self.dim ** -0.5
        for b, (n, keys) in enumerate(self.lens):
            rows = slice(at, at + n)
            at += n
            if n == 0 or (some is not None and b not in some):
                continue
            ids = torch.tensor(self.page_ids[b], dtype=torch.long, device="cuda")
            bad = torch.zeros(len(ids) * self.page, dtype=torch.bool, device="cuda")
            outside = (ids < 0) | (ids >= k_all.shape[0])
            bad = outside.repeat_interleave(self.page)[:keys]
            ids = torch.where(outside, 0, ids)
            pos = torch.arange(keys - n, keys, device="cuda")[:, None]
            key = torch.arange(keys, device="cuda")
            sees = (~bad)[None].expand(n, -1)
            if self.causal:
                sees = sees & (key <= pos)
            if self.window >= 0:
                sees = sees & (key >= pos - self.window)
            for h in range(self.q_heads):
                k = k_all[ids, h // group].reshape(-1, self.dim)[:keys]
                v = v_all[ids, h // group].reshape(-1, self.dim)[:keys]
                q = self.q[rows, h].double()
                s = (q @ k.T) * scale
                e = (self.dim + 4) * U * scale * (q.abs() @ k.abs().T)
                if self.soft_cap:
                    s = self.soft_cap * torch.tanh(s / self.soft_cap)
                    e = e + 8 * U * self.soft_cap
                s = s.masked_fill(~sees, -math.inf)
                lse = torch.logsumexp(s, 1) if keys else torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
                none = lse == -math.inf
                p = torch.exp(s - torch.where(none, 0.0, lse)[:, None])
                # Only what a row sees counts: zero times a hidden NaN is nothing.
                seen_v = torch.where(torch.isnan(v), 0.0, v)
                want = p @ seen_v
                poisoned = (sees.double() @ torch.isnan(v).double()) > 0
                score = (2 * (e + 2 * s.abs() * U).masked_fill(~sees, 0.0).amax(1) + U) if keys else torch.zeros(n, device="cuda")
                assert torch.isnan(score).any() or (score < 0.5).all()
                err = (score + keys * U)[:, None]
                bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -7) * (2.0 ** -8 + 2 * err) * (p @ seen_v.abs()) + \
                    2.0 ** -126 * (sees.double() @ seen_v.abs()) + 2.0 ** -133
                want = torch.where(poisoned | torch.isnan(lse)[:, None], math.nan, want)
                _within(self.out[rows, h], want, bound, f"{what} sequence {b} head {h} out")
                near = err[:, 0] * math.log2(math.e) + 4 * U * (lse / math.log(2)).abs()
                _within(self.lse[rows, h], lse / math.log(2), near, f"{what} sequence {b} head {h} lse")
        assert (self.out[at:] == 7).all() and (self.lse[at:] == 7).all(), f"{what}: rows of no sequence changed"


def _within(got, want, bound, what):
    got = got.double()
    same = torch.isnan(want) & torch.isnan(got) | (want == got)
    bad = ~same & ~((got - want).abs() <= bound)
    if bad.any():
        i = tuple(int(x) for x in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bound, first at {i}: got {float(got[i])!r}, want "
                             f"{float(want[i])!r}, off {float((got[i] - want[i]).abs()):.3e}, bound {float(bound[i]):.3e}")


# ---- pages: one request after another, on host lists -------------------------------------------------------------------------

class Pages:
    """The tables as Python lists, and the calls on them by their definitions."""

    def __init__(self, tables, lengths, refs, page):
        self.tables, self.lengths, self.refs, self.page = tables, lengths, refs, page
        self.width = len(tables[0])

    def used(self, s):
        return -(-min(max(self.lengths[s], 0), self.width * self.page) // self.page)

    def held(self, s):
        return [p for p in self.tables[s][:self.used(s)] if 0 <= p < len(self.refs)]

    def fork(self, pairs):
        """(status, page copies)"""
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        before = list(self.lengths)
        status, copies, named, asked = [], [], set(), 0
        for parent, child in pairs:
            known = 0 <= child < len(before)
            ok = known and child not in named and before[child] <= 0 and 0 <= parent < len(before) and before[parent] > 0
            named.add(child)
            if ok and before[parent] % self.page:
                ok = asked < len(free)
                asked += 1
            status.append(int(ok))
            if not ok:
                continue
            whole = before[parent] // self.page
            row = self.tables[parent]
            for b in range(whole):
                self.tables[child][b] = row[b]
                if 0 <= row[b] < len(self.refs):
                    self.refs[row[b]] += 1
            if before[parent] % self.page:
                page = free[asked - 1]
                self.tables[child][whole] = page
                self.refs[page] = 1
                if 0 <= row[whole] < len(self.refs):
                    copies.append((row[whole], page))
            self.lengths[child] = before[parent]
        return status, copies

    def grow(self, requests, cu):
        """(status, slots)"""
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        status, slots, named, asked = [], [], set(), 0
        for s, n in zip(requests, (b - a for a, b in zip(cu, cu[1:]))):
            ok = 0 <= s < len(self.lengths) and s not in named and self.lengths[s] + n <= self.width * self.page
            named.add(s)
            if ok:
                have = self.used(s)
                need = -(-(self.lengths[s] + n) // self.page) - have
                ok = need == 0 or asked + need <= len(free)
                taken = free[asked:asked + need]
                asked += need
            status.append(int(ok))
            if not ok:
                slots += [-1] * n
                continue
            for i, p in enumerate(taken):
                self.tables[s][have + i] = p
                self.refs[p] = 1
            for pos in range(self.lengths[s], self.lengths[s] + n):
                slots.append(self.tables[s][pos // self.page] * self.page + pos % self.page)
            self.lengths[s] += n
        return status, slots

    def free(self, requests):
        for s in requests:
            if not 0 <= s < len(self.lengths):
                continue
            for b in range(self.used(s)):
                p = self.tables[s][b]
                if 0 <= p < len(self.refs):
                    self.refs[p] -= 1
                    self.tables[s][b] = -1
            self.lengths[s] = 0

    def compact(self):
        """(live, page copies)"""
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] <= 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(len(self.tables)):
            for b in range(self.used(s)):
                self.tables[s][b] = to.get(self.tables[s][b], self.tables[s][b])
        return live, list(to.items())


def copied(pool, pairs):
    """The pool [layers, pages, ...] after one page copy after the other."""
    pool = pool.clone()
    for a, b in pairs:
        if 0 <= a < pool.shape[1] and 0 <= b < pool.shape[1]:
            pool[:, b] = pool[:, a]
    return pool
