"""The operators that stand between a layer's residual stream and its projections, as cases to time and to compare.

  norm         s = x + residual; y = s / rms(s) * weight
  norm-quant   the same row in 8 bits (e4m3) with a scale for each row or each group of its columns
  silu-quant   silu(gate) * up in 8 bits, scaled the same way, from the fused gate/up projection
  lora         y = x W^T + scale_a B_a (A_a x) + addend, a the low-rank adapter that the row's sequence names (or none)

Sizes are those of the attention and Gated DeltaNet calls beside them: one chat to 64 decode rows, ragged prompt chunks to
thousands of tokens, 8 query heads of 256 over 2 KV heads and 32 of 128 over 8. Lengths, adapters and ranks come from the
case (`lengths` seeds them), values from the seed given to prepare(). Where `own` is false, run() computes the operators in
elementary torch operations in 32 bits; where it is true it makes the library's calls.
"""
import itertools
import math
import random

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126  # a row of zeros has this scale, so that dividing by it is harmless
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f8": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f32": 4, "f8": 1, "none": 0}


def _norm(**kw):
    """A norm over `rows` rows; group < 0: not quantised, 0: one scale a row, else one scale for each `group` columns."""
    case = {"kind": "norm", "rows": 1, "dim": 1024, "x": "bf16", "residual": "bf16", "weight": "bf16", "group": -1,
            "strided": False}
    case.update(kw)
    return case


def _silu(**kw):
    case = {"kind": "silu-quant", "rows": 1, "dim": 4096, "x": "bf16", "group": 0}
    case.update(kw)
    return case


def _lora(**kw):
    """One projection over `singles` one-token sequences, then `chunks` longer ones, then `pad` rows of no sequence."""
    case = {"kind": "lora", "x": "bf16", "out": "bf16", "singles": 0, "chunks": 0, "new_lo": 2, "new_hi": 2, "pad": 0,
            "in_dim": 1024, "out_dim": 6144, "adapters": 8, "max_rank": 16, "shared": True, "addend": "none", "lengths": 1}
    case.update(kw)
    return case


def listed():
    return [
        # One chat, one token, a hybrid model's width: the smallest call there is, bound by latency.
        dict(_norm(rows=1, dim=1024), name="norm-one"),
        # A full prefill pass of 32 heads of 128, bf16 branch output onto an f32 residual stream: bound by HBM.
        dict(_norm(rows=8192, dim=4096, residual="f32"), name="norm-prefill"),
        # A decode batch whose projections take 8-bit rows.
        dict(_norm(rows=64, dim=4096, group=0), name="norm-quant-decode"),
        # A ragged prefill pass of an odd width, a scale for each 128 columns (the last group short), strided input rows.
        dict(_norm(rows=6007, dim=5000, group=128, strided=True), name="norm-quant-odd"),
        # The MLP's activation in a decode step: 48 rows of a fused gate/up projection.
        dict(_silu(rows=48, dim=12288), name="silu-quant-decode"),
        # The same in a prefill pass: bound by HBM.
        dict(_silu(rows=8192, dim=12288), name="silu-quant-prefill"),
        # One chat with an adapter, the Gated DeltaNet layer's 6,144 channels: bound by latency.
        dict(_lora(singles=1, lengths=2), name="lora-one"),
        # A decode bucket of 64 rows, 61 of them live, 24 adapters of mixed rank, the q/k/v projection of 32 over 8 heads.
        dict(_lora(singles=61, pad=3, in_dim=4096, out_dim=6144, adapters=24, max_rank=32, lengths=3), name="lora-decode"),
        # A worker step: 48 decode rows and two prompt chunks of 512, the attention output projection of 8 heads of 256
        # added onto the residual.
        dict(_lora(singles=48, chunks=2, new_lo=512, new_hi=512, in_dim=2048, out_dim=1024, addend="bf16", lengths=5),
             name="lora-mixed"),
        # Four long prompts of odd lengths, each with its adapter: bound by the matrix instructions.
        dict(_lora(chunks=4, new_lo=3500, new_hi=4096, in_dim=4096, out_dim=4096, max_rank=64, lengths=4),
             name="lora-prefill"),
        # A prefill pass over 8-bit rows and weights, as norm-quant leaves the rows: the largest product.
        dict(_lora(x="f8", chunks=5, new_lo=1000, new_hi=2048, in_dim=4096, out_dim=12288, max_rank=32, lengths=6),
             name="lora-prefill-8bit"),
        # The adapters alone, added onto the output of a product that ran elsewhere.
        dict(_lora(chunks=3, new_lo=900, new_hi=2000, in_dim=4096, out_dim=4096, shared=False, addend="bf16", lengths=7),
             name="lora-beside"),
    ]


# ---- more cases of the same ranges --------------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["norm", "norm-quant", "silu-quant", "lora", "lora", "lora", "lora-beside"])
    seed = rng.randrange(1, 1 << 20)
    if kind in ("norm", "norm-quant"):
        # Any width for the norms: half of them the multiples of 64 that models have, the others odd ones too.
        dim = 64 * _log(rng, 8, 160) if rng.random() < 0.5 else _log(rng, 300, 10000)
        x = rng.choice(["bf16", "bf16", "bf16", "f32"])
        return _norm(rows=_log(rng, 1, 8192), dim=dim, x=x, strided=rng.random() < 0.3, weight=rng.choice(["bf16", "f32"]),
                     residual=rng.choice(["bf16", "bf16", "f32", "none"]) if x == "bf16" else "f32",
                     group=-1 if kind == "norm" else rng.choice([0, 0, 128]))
    if kind == "silu-quant":
        dim = 64 * _log(rng, 16, 256) if rng.random() < 0.6 else _log(rng, 300, 14000)
        return _silu(rows=_log(rng, 1, 8192), dim=dim, x=rng.choice(["bf16", "bf16", "bf16", "f32"]),
                     group=rng.choice([0, 0, 128]))
    c = _lora(in_dim=64 * _log(rng, 8, 96), out_dim=8 * _log(rng, 64, 1600) + rng.choice([0, 0, 5]),
              adapters=_log(rng, 1, 40), max_rank=rng.choice([8, 16, 16, 32, 64]), lengths=seed,
              x=rng.choice(["bf16", "bf16", "bf16", "f8", "f8", "f32"]), addend=rng.choice(["none", "none", "bf16"]))
    if kind == "lora-beside":
        c.update(shared=False, addend="bf16", x=rng.choice(["bf16", "f8"]))
    mix = rng.choice(["singles", "singles", "chunks", "both"])
    if mix != "chunks":
        c["singles"] = _log(rng, 1, 128)
        c["pad"] = rng.choice([0, 0, 1, 7])
    if mix != "singles":
        c["chunks"] = rng.randint(1, 6)
        c["new_hi"] = _log(rng, 8, 4096 if mix == "chunks" else 1024)
        c["new_lo"] = max(2, c["new_hi"] // rng.choice([1, 4]))
    if c["x"] == "f32":  # the parity configuration: a few short sequences
        c.update(singles=min(c["singles"], 8), new_hi=min(c["new_hi"], 100), new_lo=2, out="f32", in_dim=min(c["in_dim"], 1024),
                 out_dim=min(c["out_dim"], 2048), adapters=min(c["adapters"], 4),
                 addend="f32" if c["addend"] != "none" else "none")
    elif rng.random() < 0.15:
        c["out"] = "f32"
    return c


def _cost(case):
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 5e14


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


# ---- lengths, adapters and algorithmic work --------------------------------------------------------------------------------

def _batch(case):
    """(tokens of each sequence, adapter of each sequence or -1, rank of each adapter)."""
    rng = random.Random(case["lengths"])
    n = [1] * case["singles"] + [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["chunks"])]
    # One sequence in eight has no adapter, except where there is only one sequence.
    slots = [rng.randrange(case["adapters"]) if len(n) == 1 or rng.random() >= 0.125 else -1 for _ in n]
    # Two adapters in three have the pool's full rank, the others a part of it.
    ranks = [case["max_rank"] if rng.random() < 0.67 else rng.randint(1, case["max_rank"]) for _ in range(case["adapters"])]
    return n, slots, ranks


def work(case):
    if case["kind"] == "lora":
        n, slots, ranks = _batch(case)
        t, k, m = sum(n), case["in_dim"], case["out_dim"]
        e = BYTES[case["x"]]
        low = 4 if case["x"] == "f32" else 2
        used = sum(ranks[a] for a in set(slots) if a >= 0)
        nbytes = t * k * e + t * m * (BYTES[case["out"]] + BYTES[case["addend"]]) + used * (k + m) * low
        flops = 2.0 * (k + m) * sum(c * ranks[a] for c, a in zip(n, slots) if a >= 0)
        if case["shared"]:
            nbytes += k * m * e
            flops += 2.0 * t * k * m
        return {"bytes": nbytes, "flops": flops}
    r, d = case["rows"], case["dim"]
    groups = 0 if case["group"] < 0 else 1 if case["group"] == 0 else -(-d // case["group"])
    out = BYTES[case["x"]] if case["group"] < 0 else 1
    if case["kind"] == "norm":
        return {"bytes": r * d * (BYTES[case["x"]] + 2 * BYTES[case["residual"]] + out) + 4 * r * groups, "flops": 6.0 * r * d}
    return {"bytes": r * d * (2 * BYTES[case["x"]] + out) + 4 * r * groups, "flops": 6.0 * r * d}


# ---- inputs on the GPU --------------------------------------------------------------------------------------------------

def _values(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape, std=1.0: torch.randn(shape, generator=g, device="cuda") * std


def _activations(v, rows, cols, kind):
    """Rows whose columns differ in size, some of them by a lot, as activations' do."""
    return (v(rows, cols) * torch.exp(v(cols, std=0.7))).to(TYPES[kind])


def _norm_inputs(case, v):
    r, d = case["rows"], case["dim"]
    wide = _activations(v, r, d + 24, case["x"]) if case["strided"] else _activations(v, r, d, case["x"])
    s = {"x": wide[:, :d], "weight": (1 + v(d, std=0.1)).to(TYPES[case["weight"]]), "residual": None, "residual_out": None}
    if case["residual"] != "none":
        s["residual"] = v(r, d, std=2.0).to(TYPES[case["residual"]])
        s["residual_out"] = torch.empty_like(s["residual"])
    _outputs(case, s)
    return s


def _silu_inputs(case, v):
    r, d = case["rows"], case["dim"]
    fused = _activations(v, r, 2 * d, case["x"])
    s = {"fused": fused, "gate": fused[:, :d], "up": fused[:, d:]}
    _outputs(case, s)
    return s


def _outputs(case, s):
    r, d, group = case["rows"], case["dim"], case["group"]
    s["y"] = torch.empty((r, d), dtype=TYPES[case["x"] if group < 0 else "f8"], device="cuda")
    s["scales"] = None if group < 0 else torch.empty((r, -(-d // (group or d))), device="cuda")


def _lora_inputs(case, v):
    n, slots, ranks = _batch(case)
    t, k, m, a, r = sum(n) + case["pad"], case["in_dim"], case["out_dim"], case["adapters"], case["max_rank"]
    low = torch.float32 if case["x"] == "f32" else torch.bfloat16
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"slots": i32(slots), "cu": i32(list(itertools.accumulate(n, initial=0))), "ranks": i32(ranks),
         "lora_scale": 0.5 + v(a, std=0.1),
         "lora_a": v(a, r, k, std=k ** -0.5).to(low), "lora_b": v(a, m, r, std=0.5 * r ** -0.5).to(low),
         "x_scale": None, "w_scale": None, "weight": None, "addend": None}
    if case["x"] == "f8":
        # Rows and weights in 8 bits over their whole range, with the scales that bring them back.
        x, w = v(t, k), v(m, k, std=k ** -0.5) if case["shared"] else None
        s["x"], s["x_scale"] = _to_e4m3(x)
        if w is not None:
            s["weight"], s["w_scale"] = _to_e4m3(w)
    else:
        s["x"] = v(t, k).to(TYPES[case["x"]])
        if case["shared"]:
            s["weight"] = v(m, k, std=k ** -0.5).to(TYPES[case["x"]])
    if case["addend"] != "none":
        s["addend"] = v(t, m).to(TYPES[case["addend"]])
    s["y"] = v(t, m).to(TYPES[case["out"]])  # what rows of no sequence keep
    s["before"] = s["y"].clone()
    return s


def _to_e4m3(x):
    scale = torch.clamp(x.abs().amax(1) / E4M3_MAX, min=SMALLEST_SCALE)
    return torch.clamp(x / scale[:, None], -E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _inputs(case, seed):
    v = _values(seed)
    return {"norm": _norm_inputs, "silu-quant": _silu_inputs, "lora": _lora_inputs}[case["kind"]](case, v)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["call"] = _call(case, s)
    return s


# ---- the library's calls --------------------------------------------------------------------------------------------------

def _call(case, s):
    """The call with the records and the workspace that a worker keeps: a function of no arguments."""
    import roost_amd

    session = roost_amd.OpSession()
    s["session"] = session
    if case["kind"] == "lora":
        p = roost_amd.gemm_lora_params(
            s["x"], s["weight"], s["lora_a"], s["lora_b"], s["lora_scale"], s["slots"], s["cu"], s["y"], ranks=s["ranks"],
            x_scale=s["x_scale"], w_scale=s["w_scale"], addend=s["addend"])
        ws = roost_amd.gemm_lora_workspace(session, p)
        return lambda: roost_amd.gemm_lora(session, p, ws)
    if case["kind"] == "silu-quant":
        p = roost_amd.silu_mul_quant_params(s["gate"], s["up"], s["y"], s["scales"], group_size=case["group"])
        return lambda: roost_amd.silu_mul_quant(session, p)
    if case["group"] < 0:
        p = roost_amd.add_rms_norm_params(s["x"], s["residual"], s["weight"], s["residual_out"], s["y"], eps=EPS)
        return lambda: roost_amd.add_rms_norm(session, p)
    p = roost_amd.add_rms_norm_quant_params(s["x"], s["residual"], s["weight"], s["residual_out"], s["y"], s["scales"],
                                            eps=EPS, group_size=case["group"])
    return lambda: roost_amd.add_rms_norm_quant(session, p)


# ---- the plain forms --------------------------------------------------------------------------------------------------------

def _quantised(y, group):
    """(y / scale in e4m3, scale): scale = the largest |y| of the row or of each group of its columns, over 448."""
    rows, dim = y.shape
    width = group or dim
    groups = -(-dim // width)
    cells = torch.nn.functional.pad(y, (0, groups * width - dim)).view(rows, groups, width)
    scale = torch.clamp(cells.abs().amax(2) / E4M3_MAX, min=SMALLEST_SCALE)
    q = torch.clamp(cells / scale[:, :, None], -E4M3_MAX, E4M3_MAX)
    return q.view(rows, groups * width)[:, :dim].to(torch.float8_e4m3fn), scale


def _norm_plain(case, s):
    t = s["x"].float()
    out = {}
    if s["residual"] is not None:
        t = t + s["residual"].float()
        out["residual"] = t.to(s["residual"].dtype)
    y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + EPS) * s["weight"].float()
    if case["group"] < 0:
        return dict(out, y=y.to(s["x"].dtype))
    q, scale = _quantised(y, case["group"])
    return dict(out, y=q, scales=scale)


def _silu_plain(case, s):
    g = s["gate"].float()
    q, scale = _quantised(g / (1 + torch.exp(-g)) * s["up"].float(), case["group"])
    return {"y": q, "scales": scale}


def _lora_plain(case, s):
    """Every adapter's product for every row, and zeros where the row is not the adapter's or past its rank."""
    x = s["x"].float()
    if s["x_scale"] is not None:
        x = x * s["x_scale"][:, None]
    row = torch.arange(x.shape[0], device=x.device)
    seq = torch.searchsorted(s["cu"], row.to(torch.int32), right=True) - 1
    live = seq < s["slots"].shape[0]
    slot = torch.where(live, s["slots"][torch.clamp(seq, max=s["slots"].shape[0] - 1)], -1)
    adapters, rank, k = s["lora_a"].shape
    m = s["lora_b"].shape[1]
    mine = slot[:, None] == torch.arange(adapters, device=x.device)[None, :]
    within = torch.arange(rank, device=x.device)[None, :] < s["ranks"][:, None]
    keep = mine[:, :, None] & within[None]
    u = (x @ s["lora_a"].float().view(adapters * rank, k).T).view(-1, adapters, rank)
    u = torch.where(keep, u * s["lora_scale"][None, :, None], 0.0)
    y = u.view(-1, adapters * rank) @ s["lora_b"].float().transpose(1, 2).reshape(adapters * rank, m)
    if s["weight"] is not None:
        w = s["weight"].float()
        y = y + x @ (w if s["w_scale"] is None else w * s["w_scale"][:, None]).T
    if s["addend"] is not None:
        y = y + s["addend"].float()
    return {"y": torch.where(live[:, None], y.to(s["y"].dtype), s["before"])}


def run(s):
    case = s["case"]
    if own:
        s["call"]()
        if case["kind"] == "lora":
            return {"y": s["y"]}
        out = {"y": s["y"]}
        if s.get("residual_out") is not None:
            out["residual"] = s["residual_out"]
        if s["scales"] is not None:
            out["scales"] = s["scales"]
        return out
    return {"norm": _norm_plain, "silu-quant": _silu_plain, "lora": _lora_plain}[case["kind"]](case, s)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def _scales64(y, group):
    d = y.shape[1]
    width = group or d
    tops = [y[:, c:c + width].abs().max(1).values / E4M3_MAX for c in range(0, d, width)]
    return torch.stack(tops, 1).clamp(min=SMALLEST_SCALE)


def _exact_quant(y, group):
    d = y.shape[1]
    scales = _scales64(y, group)
    of_column = torch.arange(d, device=y.device) // (group or d)
    return {"y": y / scales[:, of_column], "scales": scales}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "norm":
        t = s["x"].double()
        if s["residual"] is not None:
            t += s["residual"].double()
        y = s["weight"].double() * t / ((t ** 2).sum(1) / case["dim"] + EPS).sqrt()[:, None]
        out = {"y": y} if case["group"] < 0 else _exact_quant(y, case["group"])
        if s["residual"] is not None:
            out["residual"] = t
        return out
    if case["kind"] == "silu-quant":
        g = s["gate"].double()
        return _exact_quant(g * torch.sigmoid(g) * s["up"].double(), case["group"])
    n, slots, ranks = _batch(case)
    x = s["x"].double()
    if s["x_scale"] is not None:
        x = x * s["x_scale"].double()[:, None]
    y = s["before"].double()
    w = None if s["weight"] is None else s["weight"].double()
    if s["w_scale"] is not None:
        w = w * s["w_scale"].double()[:, None]
    live = sum(n)
    y[:live] = 0 if w is None else x[:live] @ w.T
    if s["addend"] is not None:
        y[:live] += s["addend"][:live].double()
    at = 0
    for tokens, a in zip(n, slots):
        if a >= 0:
            r = ranks[a]
            u = x[at:at + tokens] @ s["lora_a"][a, :r].double().T
            y[at:at + tokens] += s["lora_scale"][a].double() * (u @ s["lora_b"][a, :, :r].double().T)
        at += tokens
    return {"y": y}
