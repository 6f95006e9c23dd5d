"""A KV cache held in 4 bits, the attention that reads it and the pages that it lives in, as cases to time and to compare.

  write      K and V rows to 4 bits (e2m1 codes, a power-of-two scale for each 32 of a row) into their slots, and back from them
  attention  attention over such a cache: decode rows, prompt chunks on cached prefixes, both in one step
  copy       pages copied to other pages, in every layer's pools
  fork       sequences forked (whole pages shared, the last partly filled one copied), grown by a few tokens, and freed
  compact    sequences freed, and the pages that are left moved down to the pool's first ones

Sizes are those of the attention and Gated DeltaNet calls beside them: one chat to 64 decode rows, prompt chunks to thousands
of tokens, 8 query heads of 256 over 2 KV heads and 32 of 128 over 8, pages of 16 to 128 tokens. Lengths, page tables and
requests come from the case (`lengths` seeds them), values from the seed given to prepare(). Where `own` is false, run()
computes the operators in elementary torch operations; where it is true it makes the library's calls.
"""
import itertools
import math
import random

import torch

own = False

BLOCK = 32              # values that share a scale
LOW, HIGH = 7, 252      # scale bytes: 2^-120 .. 2^125; 255 marks a block that holds a NaN or an infinity
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _write(**kw):
    """`tokens` rows into slots of a pool with room for twice as many, `pad` rows of no slot among them."""
    case = {"kind": "write", "tokens": 1, "pad": 0, "kv_heads": 2, "head_dim": 256, "page": 16, "x": "bf16", "fused": False,
            "lengths": 1}
    case.update(kw)
    return case


def _attention(**kw):
    """`rows` sequences of one new token on ctx_lo..ctx_hi keys, and `chunks` of new_lo..new_hi tokens behind cached ones."""
    case = {"kind": "attention", "rows": 0, "ctx_lo": 1, "ctx_hi": 1, "chunks": 0, "new_lo": 2, "new_hi": 2, "pre_lo": 0,
            "pre_hi": 0, "q_heads": 8, "kv_heads": 2, "head_dim": 256, "page": 16, "window": -1, "soft_cap": 0.0, "csr": False,
            "lengths": 1}
    case.update(kw)
    return case


def _pages(kind, **kw):
    """A pool of `pages` pages in `layers` layers (K and V), holding `sequences` sequences of len_lo..len_hi tokens."""
    case = {"kind": kind, "layers": 6, "kv_heads": 2, "head_dim": 256, "page": 16, "pages": 1024, "sequences": 8, "len_lo": 1,
            "len_hi": 500, "count": 1, "lengths": 1}
    case.update(kw)
    return case


def listed():
    return [
        # One chat's token, one layer of a hybrid model: the smallest call, bound by latency.
        dict(_write(), name="write-one"),
        # A prefill pass of 8 KV heads, K and V read out of the fused projection, some rows of a padded batch.
        dict(_write(tokens=8181, pad=11, kv_heads=8, head_dim=128, page=64, fused=True, lengths=2), name="write-prefill"),
        # One chat, one token: bound by latency.
        dict(_attention(rows=1, ctx_lo=1500, ctx_hi=1500), name="decode-one"),
        # A full decode batch of 32 heads over 8, ragged contexts: bound by the cache's bytes.
        dict(_attention(rows=64, ctx_lo=512, ctx_hi=16000, q_heads=32, kv_heads=8, head_dim=128, lengths=3),
             name="decode-batch"),
        # Two long prompts of odd lengths on cached prefixes: bound by the matrix instructions.
        dict(_attention(chunks=2, new_lo=3500, new_hi=4096, pre_lo=1000, pre_hi=4000, q_heads=32, kv_heads=8, head_dim=128,
                        lengths=4), name="prefill-long"),
        # A worker step: 24 decode rows and two prompt chunks of 256, a hybrid model's heads, tables as the plan region has them.
        dict(_attention(rows=24, ctx_lo=300, ctx_hi=4000, chunks=2, new_lo=256, new_hi=256, pre_lo=2048, pre_hi=3000, csr=True,
                        lengths=5), name="step-mixed"),
        # Pages that an engine on the host places: a handful, in a hybrid model's six attention layers.
        dict(_pages("copy", count=5, lengths=6), name="copy-few"),
        # The same after a large preemption, 24 layers of 8 KV heads: bound by HBM.
        dict(_pages("copy", layers=24, kv_heads=8, head_dim=128, pages=3000, count=1200, lengths=7), name="copy-many"),
        # One chat answered four times over.
        dict(_pages("fork", sequences=5, count=4, lengths=8), name="fork-few"),
        # Sixteen prompts sampled eight times each, in a pool of many pages.
        dict(_pages("fork", layers=24, kv_heads=8, head_dim=128, pages=8000, sequences=144, len_hi=3000, count=128, lengths=9),
             name="fork-many"),
        # A few sequences end in a small pool.
        dict(_pages("compact", pages=600, sequences=12, count=4, lengths=10), name="compact-few"),
        # Half of a large batch ends: thousands of pages move down, in 24 layers.
        dict(_pages("compact", layers=24, kv_heads=8, head_dim=128, pages=9000, sequences=96, len_lo=200, len_hi=2400, count=48,
                    lengths=11), name="compact-many"),
    ]


# ---- more cases of the same ranges --------------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """(query heads, KV heads, head dim)"""
    group = rng.choice([1, 2, 3, 4, 4, 4, 5, 6, 8, 16])
    kv, dim = rng.choice([(1, 256), (2, 256), (4, 128), (8, 128), (8, 64), (2, 128)])
    return group * kv, kv, dim


def _draw(rng):
    kind = rng.choice(["write", "attention", "attention", "attention", "attention", "copy", "fork", "compact"])
    seed = rng.randrange(1, 1 << 20)
    q_heads, kv_heads, dim = _heads(rng)
    c = {"kv_heads": kv_heads, "head_dim": dim, "page": rng.choice([16, 16, 32, 64, 128]), "lengths": seed}
    if kind == "write":
        return _write(tokens=_log(rng, 1, 16384), pad=rng.choice([0, 0, 1, 9]), x=rng.choice(["bf16", "bf16", "f16", "f32"]),
                      fused=rng.random() < 0.5, **c)
    if kind == "attention":
        c.update(q_heads=q_heads, csr=rng.random() < 0.4, window=rng.choice([-1, -1, -1, 127, 1024]),
                 soft_cap=rng.choice([0.0, 0.0, 0.0, 30.0]))
        mix = rng.choice(["rows", "rows", "chunks", "chunks", "both"])
        if mix != "chunks":
            c.update(rows=_log(rng, 1, 64 if mix == "rows" else 24), ctx_hi=_log(rng, 16, 16000 if mix == "rows" else 4000))
            c["ctx_lo"] = max(1, c["ctx_hi"] // rng.choice([1, 4, 32]))
        if mix != "rows":
            c.update(chunks=rng.randint(1, 4), new_hi=_log(rng, 2, 4096 if mix == "chunks" else 256))
            c["new_lo"] = max(2, c["new_hi"] // rng.choice([1, 3]))
            c["pre_hi"] = rng.choice([0, _log(rng, 1, 4000)])
        return _attention(**c)
    hi = _log(rng, 20, 3000)
    n = _log(rng, 2, 160)
    c.update(layers=_log(rng, 1, 32), sequences=n, len_lo=max(1, hi // rng.choice([1, 5, 50])), len_hi=hi,
             count=rng.randint(1, max(1, n // 2)))
    c["pages"] = 2 * n * (hi // c["page"] + 2)
    if kind == "copy":
        c["count"] = _log(rng, 1, max(1, c["pages"] // 3))
    return _pages(kind, **c)


def _cost(case):
    """Of one pass in elementary operations: bytes, and the padded products of attention."""
    w = work(case)
    if case["kind"] != "attention":
        return w["bytes"] / 1e12
    n, keys = _batch(case)
    area = len(n) * max(n) * max(keys) * case["q_heads"]
    return area * (4.0 * case["head_dim"] / 5e13 + 60 / 2e12) + w["bytes"] / 5e11


def _held(case):
    """Bytes of the pools, and of what attention in elementary operations holds beside them."""
    if case["kind"] == "write":
        return 4.0 * case["tokens"] * _row_bytes(case)
    if case["kind"] == "attention":
        n, keys = _batch(case)
        return len(n) * max(keys) * (24.0 * case["kv_heads"] * case["head_dim"] + 8.0 * max(n) * case["q_heads"])
    return 2.0 * case["layers"] * case["pages"] * case["page"] * _row_bytes(case)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and _held(c) < (3e10 if c["kind"] == "attention" else 4e9):
            return c


# ---- lengths, tables, requests and algorithmic work ------------------------------------------------------------------------

def _row_bytes(case):
    """One token's K (or V) row in one layer: codes and scales."""
    return case["kv_heads"] * (case["head_dim"] // 2 + case["head_dim"] // BLOCK)


def _batch(case):
    """(new tokens, keys with them) of each sequence of an attention case."""
    rng = random.Random(case["lengths"])
    n = [1] * case["rows"] + [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["chunks"])]
    keys = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["rows"])]
    return n, keys + [c + rng.randint(case["pre_lo"], case["pre_hi"]) for c in n[case["rows"]:]]


def _seen(case, new, keys):
    """Pairs of a query and a key that it sees, in one sequence."""
    at = range(keys - new, keys)
    return sum(p + 1 if case["window"] < 0 else min(p, case["window"]) + 1 for p in at)


def _layout(case):
    """A pool in use: (pages of each sequence, tokens of each sequence). Every second page, about, is another's or free."""
    rng = random.Random(case["lengths"])
    live = case["sequences"] - (case["count"] if case["kind"] == "fork" else 0)
    lens = [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(live)]
    order = rng.sample(range(case["pages"]), case["pages"])
    tables, at = [], 0
    for n in lens:
        k = -(-n // case["page"])
        tables.append(order[at:at + k])
        at += k
    return tables, lens


def _requests(case):
    """copy: (from, to) pages; fork: (parent, child) sequences and each child's new tokens; compact: sequences that end."""
    rng = random.Random(case["lengths"] + 1)
    if case["kind"] == "copy":
        order = rng.sample(range(case["pages"]), 2 * case["count"])
        return list(zip(order[::2], order[1::2]))
    if case["kind"] == "compact":
        return rng.sample(range(case["sequences"]), case["count"])
    live = case["sequences"] - case["count"]
    return [(rng.randrange(live), live + i) for i in range(case["count"])], [rng.randint(1, 20) for _ in range(case["count"])]


def work(case):
    if case["kind"] == "write":
        # The rows in, their 4 bits out; those back in, the rows out.
        rows = 2 * case["tokens"]
        plain = case["kv_heads"] * case["head_dim"]
        back = BYTES["f32" if case["x"] == "f32" else "bf16"]
        return {"bytes": rows * (plain * (BYTES[case["x"]] + back) + 2 * _row_bytes(case)) + 16 * case["tokens"], "flops": 0.0}
    if case["kind"] == "attention":
        n, keys = _batch(case)
        seen = sum(_seen(case, a, b) for a, b in zip(n, keys))
        reach = [b if case["window"] < 0 else min(b, a + case["window"]) for a, b in zip(n, keys)]
        rows = sum(n) * case["q_heads"]
        return {"bytes": 2 * sum(reach) * _row_bytes(case) + rows * (4 * case["head_dim"] + 4),
                "flops": 4.0 * seen * case["q_heads"] * case["head_dim"]}
    page = 2 * case["layers"] * case["page"] * _row_bytes(case)
    if case["kind"] == "copy":
        return {"bytes": 2.0 * page * case["count"] + 8 * case["count"], "flops": 0.0}
    tables, lens = _layout(case)
    entries = 4.0 * sum(map(len, tables))
    if case["kind"] == "fork":
        pairs, _ = _requests(case)
        copied = sum(lens[p] % case["page"] != 0 for p, _ in pairs)
        return {"bytes": 2.0 * page * copied + sum(12 * len(tables[p]) for p, _ in pairs) + 4 * case["pages"], "flops": 0.0}
    ended = set(_requests(case))
    left = [p for i, t in enumerate(tables) if i not in ended for p in t]
    moved = sum(p >= len(left) for p in left)
    return {"bytes": 2.0 * page * moved + 2 * entries + 8 * case["pages"], "flops": 0.0}


# ---- inputs on the GPU --------------------------------------------------------------------------------------------------

def _values(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return g, lambda *shape, std=1.0: torch.randn(shape, generator=g, device="cuda") * std


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _write_inputs(case, seed):
    g, v = _values(seed)
    t, h, d, page = case["tokens"] + case["pad"], case["kv_heads"], case["head_dim"], case["page"]
    pages = -(-2 * case["tokens"] // page) + 1
    # Some of a head's dims are larger than others, as keys' are.
    x = (v(t, 3, h, d) * torch.exp(v(3, h, d, std=0.7))).to(TYPES[case["x"]])
    k, val = (x[:, 1], x[:, 2]) if case["fused"] else (x[:, 1].contiguous(), x[:, 2].contiguous())
    rng = random.Random(case["lengths"])
    slots = rng.sample(range(pages * page), case["tokens"]) + [-1] * case["pad"]
    rng.shuffle(slots)
    back = torch.float32 if case["x"] == "f32" else torch.bfloat16
    return {"k": k, "v": val, "slots": torch.tensor(slots, dtype=torch.int64, device="cuda"),
            "cache": _cache(pages, h, page, d), "k_back": torch.zeros((t, h, d), dtype=back, device="cuda"),
            "v_back": torch.zeros((t, h, d), dtype=back, device="cuda")}


def _cache(pages, heads, page, dim):
    """(K codes, K scales, V codes, V scales): codes [pages, heads, page, dim / 2], scales [pages, heads, dim / 32, page]."""
    z = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    return tuple(z(pages, heads, *s) for s in ((page, dim // 2), (dim // BLOCK, page)) * 2)


def _attention_inputs(case, seed):
    g, v = _values(seed)
    n, keys = _batch(case)
    h, d, page = case["kv_heads"], case["head_dim"], case["page"]
    blocks = [-(-k // page) for k in keys]
    pages = sum(blocks) + 3
    # Codes and scales as written rows leave them: codes that the rounding of normal values gives, scales about 2^-2.
    cache = []
    for _ in range(2):
        lane = lambda: torch.bucketize(v(pages, h, page, d // 2).abs() * 2, _thresholds())  # noqa: E731
        sign = lambda: torch.randint(0, 2, (pages, h, page, d // 2), generator=g, device="cuda") * 8  # noqa: E731
        cache += [((lane() + sign()) | (lane() + sign()) << 4).to(torch.uint8),
                  torch.randint(124, 127, (pages, h, d // BLOCK, page), generator=g, device="cuda").to(torch.uint8)]
    ids = random.Random(case["lengths"] + 1).sample(range(pages), sum(blocks))
    starts = list(itertools.accumulate(blocks, initial=0))
    table = [ids[a:b] + [-1] * (max(blocks) - b + a) for a, b in zip(starts, starts[1:])]
    q = v(sum(n), case["q_heads"], d).to(torch.bfloat16)
    return {"q": q, "cache": tuple(cache), "cu": _i32(list(itertools.accumulate(n, initial=0))), "table": _i32(table),
            "keys": _i32(keys), "ids": _i32(ids), "starts": _i32(starts),
            "last": _i32([k - (b - 1) * page for k, b in zip(keys, blocks)]), "out": torch.empty_like(q),
            "lse": torch.empty((sum(n), case["q_heads"]), device="cuda")}


def _thresholds():
    return torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")


def _pages_inputs(case, seed):
    g, _ = _values(seed)
    h, d, page, layers = case["kv_heads"], case["head_dim"], case["page"], 2 * case["layers"]
    rand = lambda *s: torch.randint(0, 256, s, dtype=torch.uint8, generator=g, device="cuda")  # noqa: E731
    s = {"codes": rand(layers, case["pages"], h * page * d // 2), "scales": rand(layers, case["pages"], h * page * d // BLOCK)}
    if case["kind"] == "copy":
        s["pairs"] = _i32(_requests(case))
        return s
    tables, lens = _layout(case)
    more = 20 // page + 2  # room to grow
    width = max(map(len, tables)) + more
    dead = case["sequences"] - len(lens)
    rows = [t + [-1] * (width - len(t)) for t in tables] + [[-1] * width] * dead
    refs = [0] * case["pages"]
    for p in itertools.chain(*tables):
        refs[p] = 1
    # One allocation, so that a pass can begin from the same tables with one copy.
    s["start"] = _i32(list(itertools.chain(*rows)) + lens + [0] * dead + refs)
    s["now"] = s["start"].clone()
    a, b = width * case["sequences"], (width + 1) * case["sequences"]
    s.update(tables=s["now"][:a].view(-1, width), lens=s["now"][a:b], refs=s["now"][b:])
    if case["kind"] == "compact":
        s.update(ended=_i32(_requests(case)), live=_i32([0]))
        return s
    pairs, new = _requests(case)
    cu = list(itertools.accumulate(new, initial=0))
    s.update(pairs=_i32(pairs), children=_i32([c for _, c in pairs]), cu=_i32(cu), forked=_i32([0] * len(pairs)),
             grown=_i32([0] * len(pairs)), slots=torch.zeros(cu[-1], dtype=torch.int64, device="cuda"))
    return s


INPUTS = {"write": _write_inputs, "attention": _attention_inputs, "copy": _pages_inputs, "fork": _pages_inputs,
          "compact": _pages_inputs}


def prepare(case, seed):
    s = INPUTS[case["kind"]](case, seed)
    s["case"] = case
    if own:
        s["call"] = _call(case, s)
    return s


# ---- the library's calls --------------------------------------------------------------------------------------------------

def _call(case, s):
    """The calls with the records and the workspace that a worker keeps: a function of no arguments."""
    import roost_amd

    session = roost_amd.OpSession()
    s["session"] = session
    page = case["page"]
    if case["kind"] == "write":
        into = roost_amd.cache_f4_params(s["k"], s["v"], s["cache"], s["slots"])
        back = roost_amd.cache_f4_params(s["k_back"], s["v_back"], s["cache"], s["slots"])

        def write():
            roost_amd.cache_write_f4(session, into)
            roost_amd.cache_read_f4(session, back)
        return write
    if case["kind"] == "attention":
        n, keys = _batch(case)
        tables = dict(kv_indptr=s["starts"], kv_indices=s["ids"], kv_last_page_len=s["last"]) if case["csr"] else \
            dict(block_tables=s["table"], kv_lens=s["keys"])
        p = roost_amd.paged_attention_f4_params(s["q"], s["out"], s["cache"], s["cu"], lse=s["lse"], max_q_len=max(n),
                                                max_kv_len=max(keys), window_left=case["window"], soft_cap=case["soft_cap"],
                                                **tables)
        ws = roost_amd.paged_attention_f4_workspace(session, p)
        return lambda: roost_amd.paged_attention_f4(session, p, ws)
    pools = [s["codes"], s["scales"]]
    if case["kind"] == "copy":
        p = roost_amd.cache_copy_params(pools, s["pairs"])
        return lambda: roost_amd.cache_copy(session, p)
    state = dict(block_tables=s["tables"], lengths=s["lens"], refs=s["refs"], page_size=page)
    if case["kind"] == "compact":
        free = roost_amd.cache_free_params(s["ended"], **state)
        p = roost_amd.cache_compact_params(pools, s["live"], **state)
        ws = roost_amd.cache_pages_workspace(session, p)

        def compact():
            s["now"].copy_(s["start"])
            roost_amd.cache_free(session, free)
            roost_amd.cache_compact(session, p, ws)
        return compact
    free = roost_amd.cache_free_params(s["children"], **state)
    fork = roost_amd.cache_fork_params(pools, s["pairs"], s["forked"], **state)
    grow = roost_amd.cache_grow_params(s["children"], s["cu"], s["slots"], s["grown"], **state)
    ws = roost_amd.cache_pages_workspace(session, fork)

    def generations():
        roost_amd.cache_free(session, free)
        roost_amd.cache_fork(session, fork, ws)
        roost_amd.cache_grow(session, grow, ws)
    return generations


# ---- the plain forms --------------------------------------------------------------------------------------------------------

def _to_f4(x):
    """(codes 0..15 [..., dim], scale bytes [..., dim / 32]) of rows [..., dim] in 32 bits.

    The scale is the smallest power of two that leaves the block's largest magnitude at 7 or below, so that nothing is off
    by more than one, half the distance of the grid's last two values."""
    cells = x.unflatten(-1, (-1, BLOCK))
    bits = cells.abs().amax(-1).view(torch.int32)
    byte = torch.clamp((bits >> 23) + ((bits & 0x7FFFFF) > 0x600000).int() - 2, LOW, HIGH)
    byte = torch.where(cells.isfinite().all(-1), byte, 255)
    r = torch.where(byte[..., None] == 255, 0.0, cells.abs() / _scale(byte)[..., None])
    ties_down = torch.tensor([0.25, 1.25, 2.5, 5.0], device=x.device)
    ties_up = torch.tensor([0.75, 1.75, 3.5], device=x.device)
    code = torch.bucketize(r, ties_down) + torch.bucketize(r, ties_up, right=True)
    return (code + 8 * torch.signbit(cells).int()).flatten(-2), byte


def _scale(byte):
    """The power of two that a scale byte stands for; NaN for 255."""
    b = byte.int()
    return torch.where(b == 255, math.nan, (b << 23).view(torch.float32))


def _from_f4(codes, scales):
    """Values [..., tokens, dim] in 32 bits of packed codes [..., tokens, dim / 2] and scale bytes [..., dim / 32, tokens]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    return grid[c] * _scale(scales).transpose(-1, -2).repeat_interleave(BLOCK, -1)


def _write_plain(case, s):
    page = case["page"]
    kept = torch.nonzero(s["slots"] >= 0).flatten()
    at, off = s["slots"][kept] // page, s["slots"][kept] % page
    out = {}
    for name, x, codes, scales in (("k", s["k"], *s["cache"][:2]), ("v", s["v"], *s["cache"][2:])):
        code, byte = _to_f4(x[kept].float())
        codes[at, :, off] = (code[..., ::2] | code[..., 1::2] << 4).to(torch.uint8)
        scales[at, :, :, off] = byte.to(torch.uint8)
        back = s[name + "_back"]
        back[kept] = _from_f4(codes[at, :, off][:, :, None], scales[at, :, :, off][..., None])[:, :, 0].to(back.dtype)
        out[name] = back
    return out


def _attention_plain(case, s):
    """Every sequence padded to the longest: [sequences, KV heads, new tokens x group, keys]."""
    n, keys = s["cu"][1:] - s["cu"][:-1], s["keys"]
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    group, batch = case["q_heads"] // h, n.shape[0]
    table = s["table"].clamp(min=0).long()
    longest = table.shape[1] * page
    most = max(_batch(case)[0])
    k, v = (_from_f4(codes[table], scales[table]).transpose(1, 2).reshape(batch, h, longest, d)
            for codes, scales in (s["cache"][:2], s["cache"][2:]))
    key = torch.arange(longest, device=n.device)
    v = torch.where((key < keys[:, None])[:, None, :, None], v, 0.0)
    row = torch.arange(most, device=n.device)
    token = (s["cu"][:-1, None] + row).clamp(max=s["q"].shape[0] - 1).long()  # [batch, most]
    live = row < n[:, None]
    q = s["q"][token].float().view(batch, most, h, group, d).permute(0, 2, 1, 3, 4).reshape(batch, h, most * group, d)
    score = (q @ k.transpose(2, 3).contiguous()) * d ** -0.5
    if case["soft_cap"]:
        score = case["soft_cap"] * torch.tanh(score / case["soft_cap"])
    pos = keys[:, None] - n[:, None] + row  # [batch, most]
    sees = (key <= pos[:, :, None]) & (key < keys[:, None, None])
    if case["window"] >= 0:
        sees &= key >= pos[:, :, None] - case["window"]
    score = score.view(batch, h, most, group, longest).masked_fill(~sees[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    p = (p / total.clamp(min=1e-38)).view(batch, h, most * group, longest)
    y = (p @ v).view(batch, h, most, group, d).permute(0, 2, 1, 3, 4)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 2, 1, 3) / math.log(2)
    return {"out": y[live].reshape(-1, case["q_heads"], d).to(torch.bfloat16), "lse": lse[live].reshape(-1, case["q_heads"])}


def _free_plain(s, slots, page):
    slots = slots.long()
    used = torch.arange(s["tables"].shape[1], device=slots.device) < -(-s["lens"][slots] // page)[:, None]
    rows = s["tables"][slots]
    s["refs"].index_add_(0, rows[used].long(), torch.full_like(rows[used], -1))
    s["tables"][slots] = torch.where(used, -1, rows)
    s["lens"][slots] = 0


def _give(s, need):
    """The pages that requests for `need` pages each are given, in their order, lowest first: [sum(need)]."""
    return torch.nonzero(s["refs"] == 0).flatten()[:int(need.sum())]


def _fork_plain(case, s):
    page = case["page"]
    _free_plain(s, s["children"], page)
    parent, child = s["pairs"].long().unbind(1)
    length = s["lens"][parent]
    whole, part = length // page, length % page != 0
    width = s["tables"].shape[1]
    column = torch.arange(width, device=length.device)
    new = _give(s, part)
    given = torch.full_like(parent, -1).masked_scatter(part, new)
    rows = s["tables"][parent]
    shared = rows[column < whole[:, None]].long()
    old = rows[part, whole[part].long()].long()
    s["refs"].index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    s["refs"][new] = 1
    last = (column == whole[:, None]) & part[:, None]
    s["tables"][child] = torch.where(last, given[:, None].int(), torch.where(column <= whole[:, None], rows, -1))
    s["lens"][child] = length
    for pool in (s["codes"], s["scales"]):
        pool[:, new] = pool[:, old]
    s["forked"].fill_(1)
    # Grown by a few tokens.
    add = s["cu"][1:] - s["cu"][:-1]
    have, want = -(-length // page), -(-(length + add) // page)
    rows = s["tables"][child]
    fresh = (column >= have[:, None]) & (column < want[:, None])
    taken = _give(s, want - have)
    rows.masked_scatter_(fresh, taken.int())
    s["refs"][taken] = 1
    s["tables"][child] = rows
    s["lens"][child] = length + add
    of = torch.repeat_interleave(torch.arange(len(add), device=add.device), add)
    pos = (length - s["cu"][:-1])[of] + torch.arange(len(of), device=add.device)
    s["slots"].copy_(rows[of, pos // page].long() * page + pos % page)
    s["grown"].fill_(1)


def _compact_plain(case, s):
    s["now"].copy_(s["start"])
    _free_plain(s, s["ended"], case["page"])
    used = s["refs"] > 0
    live = used.sum()
    page = torch.arange(len(used), device=used.device)
    holes, movers = torch.nonzero(~used & (page < live)).flatten(), torch.nonzero(used & (page >= live)).flatten()
    for pool in (s["codes"], s["scales"]):
        pool[:, holes] = pool[:, movers]
    s["refs"][holes] = s["refs"][movers]
    s["refs"][movers] = 0
    to = page.int()
    to[movers] = holes.int()
    s["tables"].copy_(torch.where(s["tables"] >= 0, to[s["tables"].clamp(min=0).long()], -1))
    s["live"].copy_(live)


def _copy_plain(case, s):
    src, dst = s["pairs"].long().unbind(1)
    for pool in (s["codes"], s["scales"]):
        pool[:, dst] = pool[:, src]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        s["call"]()
        if kind == "write":
            return {"k": s["k_back"], "v": s["v_back"]}
        if kind == "attention":
            return {"out": s["out"], "lse": s["lse"]}
    elif kind in ("write", "attention"):
        return {"write": _write_plain, "attention": _attention_plain}[kind](case, s)
    else:
        {"copy": _copy_plain, "fork": _fork_plain, "compact": _compact_plain}[kind](case, s)
    return {k: s[k] for k in ("codes", "scales", "now", "slots", "forked", "grown", "live") if k in s}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] not in ("write", "attention"):
        return None  # whole numbers
    s = INPUTS[case["kind"]](case, seed)
    if case["kind"] == "write":
        return {name: _exact_f4(s[name].double(), s["slots"] >= 0) for name in ("k", "v")}
    n, keys = _batch(case)
    h, d, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["q_heads"] // h
    outs, lses = [], []
    at = 0
    for b, (new, total) in enumerate(zip(n, keys)):
        pages = s["table"][b, :-(-total // page)].long()
        pos = torch.arange(total - new, total, device="cuda").repeat_interleave(group)[:, None]
        key = torch.arange(total, device="cuda")
        hidden = key > pos
        if case["window"] >= 0:
            hidden |= key < pos - case["window"]
        out, lse = [], []
        for head in range(h):
            k, v = (_exact_values(codes[pages, head], scales[pages, head])[:total]
                    for codes, scales in (s["cache"][:2], s["cache"][2:]))
            q = s["q"][at:at + new, head * group:(head + 1) * group].double().reshape(-1, d)
            score = q @ k.T / math.sqrt(d)
            if case["soft_cap"]:
                score = case["soft_cap"] * torch.tanh(score / case["soft_cap"])
            score[hidden] = -math.inf
            log_sum = torch.logsumexp(score, 1)
            out.append((torch.exp(score - log_sum[:, None]) @ v).view(new, group, d))
            lse.append((log_sum / math.log(2)).view(new, group))
        outs.append(torch.cat(out, 1))
        lses.append(torch.cat(lse, 1))
        at += new
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_values(codes, scales):
    """[tokens, dim] of one head's pages: codes [pages, page, dim / 2], scales [pages, dim / 32, page]."""
    lo, hi = codes.long() % 16, codes.long() // 16
    c = torch.stack((lo, hi), 3).reshape(*codes.shape[:2], -1)
    size, sign = c % 8, 1 - 2 * (c // 8)
    # e2m1: an exponent of two bits and a mantissa of one, no exponent below 1.
    value = torch.where(size < 2, 0.5 * size, (1 + 0.5 * (size % 2)) * torch.exp2((size // 2 - 1).double()))
    scale = torch.exp2(scales.double() - 127)  # exact, which pow() is not
    return (sign * value * scale.transpose(1, 2).repeat_interleave(BLOCK, 2)).flatten(0, 1)


def _exact_f4(x, kept):
    """The nearest of the grid's values, ties to the even code, times the block's scale; zeros where no slot was named."""
    cells = x.view(*x.shape[:-1], -1, BLOCK)
    top = cells.abs().amax(-1, keepdim=True)
    # The smallest power of two with top <= 7 * scale, within its range.
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 7))
    scale = torch.exp2(e.clamp(LOW - 127, HIGH - 127))
    r = cells.abs() / scale
    step = torch.exp2(torch.floor(torch.log2(r.clamp(min=1.0))).clamp(max=2.0) - 1)
    y = (torch.round(r / step) * step).clamp(max=6.0) * scale * torch.sign(cells)  # round() takes ties to even
    return torch.where(kept[:, None, None], y.view(x.shape), 0.0)
