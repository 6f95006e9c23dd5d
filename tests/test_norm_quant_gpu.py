"""AddRmsNorm, AddRmsNormQuant and SiluMulQuant on the GPU through the C ABI, against their definitions in 64 bits; the
bounds are derived in fused_cases.py."""
import pytest
import torch

import fused_cases as fc
import roost_amd
from fused_cases import BF16, F32, F8

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _values(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda") * std


def _norm_case(seed, rows, dim, x=BF16, res=BF16, w=BF16, gap=0):
    v = _values(seed)
    wide = (v(rows, dim + gap) * torch.exp(v(dim + gap, std=0.7))).to(x)
    residual = None if res is None else v(rows, dim + gap, std=2.0).to(res)[:, :dim]
    return wide[:, :dim], residual, (1 + v(dim, std=0.1)).to(w)


# rows, dim, input, residual, weight, columns between rows
NORMS = [
    (1, 1024, BF16, BF16, BF16, 0),
    (1, 1, BF16, BF16, BF16, 0),          # one column: y = +-weight
    (3, 7, BF16, F32, F32, 0),            # less than one vector
    (5, 9, F32, F32, BF16, 3),            # one vector and one column, rows at odd addresses
    (4, 511, BF16, BF16, F32, 1),
    (2, 2049, BF16, None, BF16, 0),       # no residual; more than one vector a thread
    (64, 4096, BF16, BF16, BF16, 0),
    (33, 5000, BF16, F32, BF16, 24),      # strided rows
    (7, 12288, F32, F32, F32, 0),
    (3, 16385, BF16, BF16, BF16, 0),      # four vectors a thread, odd rows
    (2, 32768, F32, BF16, BF16, 0),       # the widest row
    (1000, 640, BF16, BF16, BF16, 0),
]


@pytest.mark.parametrize("rows,dim,x,res,w,gap", NORMS)
def test_add_rms_norm(session, rows, dim, x, res, w, gap):
    xs, residual, weight = _norm_case(rows + dim, rows, dim, x, res, w, gap)
    y = torch.full((rows, dim + gap), 7.0, device="cuda", dtype=x)
    ro = torch.full((rows, dim + gap), 7.0, device="cuda", dtype=res or x)
    roost_amd.add_rms_norm(session, roost_amd.add_rms_norm_params(xs, residual, weight, ro[:, :dim], y[:, :dim], eps=EPS))
    s, want = fc.norm64(xs, residual, weight, EPS)
    fc.assert_within(y[:, :dim], want, fc.rounded_bound(want, x, fc.NORM * want.abs()), "y")
    sum32 = xs.float() if residual is None else xs.float() + residual.float()
    assert torch.equal(ro[:, :dim], sum32.to(ro.dtype))
    assert (y[:, dim:] == 7).all() and (ro[:, dim:] == 7).all()  # what lies between the rows


@pytest.mark.parametrize("rows,dim,x,res,w,gap", NORMS)
@pytest.mark.parametrize("group", [0, 128])
def test_add_rms_norm_quant(session, rows, dim, x, res, w, gap, group):
    xs, residual, weight = _norm_case(rows + dim + 1, rows, dim, x, res, w, gap)
    cells = 1 if group == 0 else -(-dim // group)
    y = torch.zeros((rows, dim + gap), device="cuda", dtype=F8)
    scales = torch.full((rows, cells), 7.0, device="cuda")
    ro = None if residual is None else torch.empty_like(residual)
    roost_amd.add_rms_norm_quant(session, roost_amd.add_rms_norm_quant_params(
        xs, residual, weight, ro, y[:, :dim], scales, eps=EPS, group_size=group))
    _, want = fc.norm64(xs, residual, weight, EPS)
    fc.assert_quantised(y[:, :dim], scales, want, group, fc.NORM, f"quant {rows}x{dim} group {group}")
    assert (y[:, dim:].float() == 0).all()
    if residual is not None:
        assert torch.equal(ro, (xs.float() + residual.float()).to(ro.dtype))


@pytest.mark.parametrize("group", [16, 32, 64, 256, 512])
def test_group_sizes(session, group):
    xs, residual, weight = _norm_case(group, 9, 1000)
    y = torch.empty((9, 1000), device="cuda", dtype=F8)
    scales = torch.empty((9, -(-1000 // group)), device="cuda")
    roost_amd.add_rms_norm_quant(session, roost_amd.add_rms_norm_quant_params(xs, residual, weight, None, y, scales, eps=EPS,
                                                                              group_size=group))
    _, want = fc.norm64(xs, residual, weight, EPS)
    fc.assert_quantised(y, scales, want, group, fc.NORM, f"group {group}")


@pytest.mark.parametrize("rows,dim,x,group", [
    (1, 1, BF16, 0), (3, 5, F32, 0), (48, 12288, BF16, 0), (7, 2909, BF16, 0), (5, 4097, F32, 128), (300, 1792, BF16, 128),
    (2, 32768, BF16, 0), (2, 32767, F32, 512)])
def test_silu_mul_quant(session, rows, dim, x, group):
    v = _values(rows + dim)
    fused = (v(rows, 2 * dim) * 3).to(x)
    gate, up = fused[:, :dim], fused[:, dim:]
    y = torch.empty((rows, dim), device="cuda", dtype=F8)
    scales = torch.empty((rows, 1 if group == 0 else -(-dim // group)), device="cuda")
    roost_amd.silu_mul_quant(session, roost_amd.silu_mul_quant_params(gate, up, y, scales, group_size=group))
    fc.assert_quantised(y, scales, fc.silu64(gate, up), group, fc.SILU, f"silu {rows}x{dim}")


def test_in_place(session):
    """output over the input and residual_out over the residual, and the other way round, give the same bits."""
    xs, residual, weight = _norm_case(3, 21, 1500)
    y, ro = torch.empty_like(xs), torch.empty_like(residual)
    roost_amd.add_rms_norm(session, roost_amd.add_rms_norm_params(xs, residual, weight, ro, y, eps=EPS))
    for a, b in ((0, 1), (1, 0)):
        bufs = [xs.clone(), residual.clone()]
        roost_amd.add_rms_norm(session, roost_amd.add_rms_norm_params(bufs[0], bufs[1], weight, bufs[b], bufs[a], eps=EPS))
        assert torch.equal(bufs[a], y) and torch.equal(bufs[b], ro)


def test_rows_do_not_depend_on_each_other(session):
    xs, residual, weight = _norm_case(4, 50, 3000)
    y = torch.empty_like(xs)
    roost_amd.add_rms_norm(session, roost_amd.add_rms_norm_params(xs, residual, weight, None, y, eps=EPS))
    one = torch.empty_like(xs[:1])
    for r in (0, 17, 49):
        roost_amd.add_rms_norm(session, roost_amd.add_rms_norm_params(xs[r:r + 1], residual[r:r + 1], weight, None, one,
                                                                      eps=EPS))
        assert torch.equal(one, y[r:r + 1])


def test_zero_and_non_finite_cells(session):
    """A row of zeros: zero codes and the smallest scale. Cells with a NaN or an infinity mark themselves, no others."""
    gate = torch.ones((4, 256), device="cuda", dtype=F32)
    up = torch.ones((4, 256), device="cuda", dtype=F32) * 3
    gate[0] = 0
    up[1, 5] = float("nan")
    up[2, 200] = float("inf")
    y = torch.empty((4, 256), device="cuda", dtype=F8)
    scales = torch.empty((4, 2), device="cuda")
    roost_amd.silu_mul_quant(session, roost_amd.silu_mul_quant_params(gate, up, y, scales, group_size=128))
    codes, s = y.float().cpu(), scales.cpu()
    assert (codes[0] == 0).all() and (s[0] == 2.0 ** -126).all()
    assert torch.isnan(codes[1, :128]).all() and torch.isnan(s[1, 0])
    assert (codes[1, 128:] == 448).all() and torch.isfinite(s[1, 1])
    assert s[2, 1] == float("inf") and torch.isnan(codes[2, 200])
    assert (codes[2, 128:200] == 0).all() and (codes[2, :128] == 448).all()
    # The norm of a row with an infinity is NaN throughout (its root is infinite), of one of zeros is zero.
    x = torch.zeros((2, 300), device="cuda", dtype=BF16)
    x[0, 7] = float("inf")
    out = torch.empty_like(x)
    w = torch.ones(300, device="cuda", dtype=BF16)
    roost_amd.add_rms_norm(session, roost_amd.add_rms_norm_params(x, None, w, None, out, eps=EPS))
    assert torch.isnan(out[0, 7]) and (out[0, :7] == 0).all() and (out[1] == 0).all()


def test_every_code_rounds_to_nearest_even(session):
    """One cell whose largest value is 448, so the scale is 1 and each other value is rounded as it stands: every e4m3
    value, every midpoint between two of them (ties to even) and their f32 neighbours."""
    codes = torch.arange(127, dtype=torch.uint8).view(F8).float()  # 0 .. 448, the finite positive codes in order
    mids = (codes[:-1] + codes[1:]) / 2
    near = torch.cat([codes, mids, torch.nextafter(mids, mids * 0), torch.nextafter(mids, mids * 2)])
    vals = torch.cat([near, -near])
    dim = vals.numel()
    # silu(gate) * up with a gate far on the right: silu(64) = 64 / (1 + e^-64) = 64 in f32.
    gate = torch.full((1, dim), 64.0, device="cuda")
    up = (vals / 64).cuda()[None]
    y = torch.empty((1, dim), device="cuda", dtype=F8)
    scales = torch.empty((1, 1), device="cuda")
    roost_amd.silu_mul_quant(session, roost_amd.silu_mul_quant_params(gate, up, y, scales))
    assert scales.item() == 1.0
    assert torch.equal(y.cpu().float()[0], vals.to(F8).float())


@pytest.mark.parametrize("top", [1.0, 3.3, 447.9, 12345.678, 1e-3, 7e-30, 2.5e-36, 6e-36, 3e33])
def test_codes_are_quotients_by_the_scale(session, top):
    """At scales that are no powers of two: the f32 quotient of each value and the scale, rounded to nearest even, bit for bit.
    Every e4m3 value and every midpoint between two of them times the scale, and the f32 neighbours of those; a
    product by the scale's reciprocal gives some of them the other code."""
    codes = torch.arange(127, dtype=torch.uint8).view(F8).float()
    mids = (codes[:-1] + codes[1:]) / 2
    near = torch.cat([codes, mids]) * (torch.tensor(top) / 448)
    scale = (torch.tensor(top) / 448).clamp(min=2.0 ** -126)
    near = torch.cat([near] + [torch.nextafter(near, near * k) for k in (0, 2)]).clamp(max=top)
    vals = torch.cat([torch.tensor([top]), near, -near])
    up = vals / 64  # silu(64) = 64 in f32
    vals = up * 64
    y = torch.empty((1, vals.numel()), device="cuda", dtype=F8)
    scales = torch.empty((1, 1), device="cuda")
    gate = torch.full_like(y, 64.0, dtype=F32)
    roost_amd.silu_mul_quant(session, roost_amd.silu_mul_quant_params(gate, up.cuda()[None], y, scales))
    assert scales.cpu().item() == scale.item()
    assert torch.equal(y.cpu().float()[0], (vals / scale).to(F8).float())


def test_graph_replays(session):
    """Captured once, replayed with other inputs and eager work in between."""
    xs, residual, weight = _norm_case(8, 40, 2000)
    y, scales = torch.empty((40, 2000), device="cuda", dtype=F8), torch.empty((40, 1), device="cuda")
    ro = torch.empty_like(residual)
    stream = torch.cuda.Stream()
    s = roost_amd.OpSession(session.lib, device=0, stream=stream)
    p = roost_amd.add_rms_norm_quant_params(xs, residual, weight, ro, y, scales, eps=EPS)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        roost_amd.add_rms_norm_quant(s, p)
    for k in range(4):
        xs.copy_(_norm_case(100 + k, 40, 2000)[0])
        y.view(torch.uint8).fill_(1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, got_scales = y.clone(), scales.clone()
        roost_amd.add_rms_norm_quant(session, p)
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.uint8), y.view(torch.uint8)) and torch.equal(got_scales, scales)
        _, want = fc.norm64(xs, residual, weight, EPS)
        fc.assert_quantised(got, got_scales, want, 0, fc.NORM, f"replay {k}")
    s.close()
