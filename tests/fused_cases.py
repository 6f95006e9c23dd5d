"""Inputs and 64-bit definitions for the fused ops between the residual stream and the projections, and the error bounds
their tests hold the kernels to.

Bounds. A rounding to bf16 is off by at most 2^-8 of the value, to f32 by 2^-24, to e4m3 by 2^-4 (or 2^-10, half its smallest
step, below 2^-6).
  * A norm row in f32: the sum of squares is at most 32 fused multiply-adds in a thread, 6 steps over a wavefront and 16
    over a workgroup; mean, root, reciprocal and the products by it and by the weight are 6 more roundings, the sum with the
    residual one: fewer than 64 roundings, NORM = 64 * 2^-24 = 2^-18 of the value.
  * SiLU in f32: exp's argument times log2(e) is off by 2^-24 |x| / ln 2, so e^-x by 2^-24 |x| and a few ulp; the sigmoid takes
    that over by at most e^-x / (1 + e^-x) <= 1. With |x| <= 64 in these inputs: 80 * 2^-24 < 2^-17 of the value.
  * A product of `n` terms in f32 sums: n additions, each off by at most 2^-23 of the sum of the terms' magnitudes (2^-23, not
    2^-24: nothing says that a matrix instruction rounds its inner sums to nearest).
"""
import torch

BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
NORM, SILU = 2.0 ** -18, 2.0 ** -17
ADD = 2.0 ** -23
PRODUCTS = 2.0 ** -10


def rounded_bound(y, dtype, more):
    """Off by `more` (an absolute bound before the rounding) and one rounding to dtype."""
    return more + HALF[dtype] * (y.abs() + more)


def assert_within(got, want, bound, what):
    got, want, bound = got.double(), want.double(), bound.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs()
    bad = off > bound
    if bad.any():
        i = tuple(int(k) for k in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bound, first at {i}: got {float(got[i])!r}, "
                             f"want {float(want[i])!r}, off {float(off[i]):.3e}, bound {float(bound[i]):.3e}")


def norm64(x, residual, weight, eps):
    """(s, y) of AddRmsNorm in 64 bits."""
    s = x.double() if residual is None else x.double() + residual.double()
    return s, s / torch.sqrt(s.square().mean(1, keepdim=True) + eps) * weight.double()


def silu64(gate, up):
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def cells64(y, group):
    """Every element's scale, and the scales [rows, cells]."""
    dim = y.shape[1]
    width = group or dim
    scales = torch.stack([y[:, c:c + width].abs().amax(1) for c in range(0, dim, width)], 1) / 448
    scales = scales.clamp(min=2.0 ** -126)
    return scales[:, torch.arange(dim, device=y.device) // width], scales


def assert_quantised(codes, scales, y, group, err, what):
    """Codes and scales of the 64-bit values y that the kernel has within err (relative): each scale within err of its
    own, each code the rounding of some value within 2 err of y / scale (both the value and the scale are off), so
    equal wherever that interval rounds to one code."""
    each, want = cells64(y, group)
    assert_within(scales, want, (err + 2.0 ** -22) * want, what + " scales")
    ratio = y / each
    step = 2 * err + 2.0 ** -21
    lo = (ratio * (1 - step)).clamp(-448, 448).float().to(F8).float()
    hi = (ratio * (1 + step)).clamp(-448, 448).float().to(F8).float()
    got = codes.float()
    bad = (got != lo) & (got != hi)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} codes are no rounding of their value"
    assert (lo == hi).double().mean() > 0.99  # the check above has teeth


class Lora:
    """One GemmLora call's inputs. lens: tokens of each sequence; slots: each one's adapter."""

    def __init__(self, seed, lens, slots, *, in_dim, out_dim, adapters=4, max_rank=16, ranks=None, x=BF16, out=BF16,
                 shared=True, addend=None, pad=0, x_gap=0, y_gap=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        v = lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda") * std  # noqa: E731
        self.lens, self.slots, self.tokens = lens, slots, sum(lens) + pad
        t = self.tokens
        self.low = F32 if x == F32 else BF16
        self.x_scale = self.w_scale = self.weight = self.addend = None
        wide = v(t, in_dim + x_gap)
        if x == F8:
            self.x_scale = 0.5 + torch.rand(t, generator=g, device="cuda")
            wide = (wide * 40).clamp(-448, 448)
        self.x = wide.to(x)[:, :in_dim]
        if shared:
            w = v(out_dim, in_dim, std=in_dim ** -0.5)
            if x == F8:
                self.w_scale = (0.5 + torch.rand(out_dim, generator=g, device="cuda")) / 64
                w = (w * 64).clamp(-448, 448)
            self.weight = w.to(x)
        self.lora_a = v(max(adapters, 1), max_rank, in_dim, std=in_dim ** -0.5).to(self.low)
        self.lora_b = v(max(adapters, 1), out_dim, max_rank, std=max(max_rank, 1) ** -0.5).to(self.low)
        self.lora_scale = 0.5 + torch.rand(max(adapters, 1), generator=g, device="cuda")
        self.adapters, self.max_rank = adapters, max_rank
        self.ranks_h = [max_rank] * adapters if ranks is None else ranks
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        self.ranks = None if ranks is None else i32(ranks)
        self.slots_d = i32(slots)
        self.cu = i32([sum(lens[:i]) for i in range(len(lens) + 1)])
        if adapters == 0:
            self.lora_a = self.lora_b = self.lora_scale = None
        if addend is not None:
            self.addend = v(t, out_dim + y_gap).to(addend)[:, :out_dim]
        self.y = v(t, out_dim + y_gap).to(out)[:, :out_dim]
        self.before = self.y.clone()

    def params(self, **kw):
        import roost_amd

        args = dict(ranks=self.ranks, x_scale=self.x_scale, w_scale=self.w_scale, addend=self.addend)
        args.update(kw)
        return roost_amd.gemm_lora_params(self.x, self.weight, self.lora_a, self.lora_b, self.lora_scale,
                                          None if self.lora_a is None else self.slots_d, self.cu, self.y, **args)

    def want(self):
        """(values, bound) in 64 bits of the live rows."""
        x = self.x.double()
        if self.x_scale is not None:
            x = x * self.x_scale.double()[:, None]
        live, out_dim = sum(self.lens), self.y.shape[1]
        y = torch.zeros((live, out_dim), dtype=torch.float64, device="cuda")
        size = torch.zeros_like(y)   # sums of magnitudes that f32 additions run over
        low = torch.zeros_like(y)    # those of the low-rank rows, which bf16 rounds once
        cut = 0.0
        terms = x.shape[1] + self.max_rank + 16
        if self.weight is not None:
            w = self.weight.double()
            if self.w_scale is not None:
                w = w * self.w_scale.double()[:, None]
            y += x[:live] @ w.T
            size += x[:live].abs() @ w.abs().T
            if self.x_scale is not None and self.y.dtype == BF16:
                eights = [v.abs().reshape(v.shape[0], -1, 8).amax(2) for v in (x[:live], w)]
                cut = PRODUCTS * (eights[0] @ eights[1].T)
        at = 0
        for n, a in zip(self.lens, self.slots):
            if n and self.lora_a is not None and 0 <= a < self.adapters:
                r = min(max(self.ranks_h[a], 0), self.max_rank)
                la, lb = self.lora_a[a, :r].double(), self.lora_b[a, :, :r].double()
                rows = x[at:at + n]
                scale = self.lora_scale[a].double()
                u = scale * (rows @ la.T)
                y[at:at + n] += u @ lb.T
                size[at:at + n] += scale * ((rows.abs() @ la.abs().T) @ lb.abs().T)
                low[at:at + n] += u.abs() @ lb.abs().T
            at += n
        if self.addend is not None:
            y += self.addend[:live].double()
            size += self.addend[:live].double().abs()
        more = terms * ADD * size + cut
        if self.low == BF16:
            more = more + 2.0 ** -8 * (low + more)
        return y, rounded_bound(y, self.y.dtype, more)

    def check(self, what=""):
        y, bound = self.want()
        live = sum(self.lens)
        assert_within(self.y[:live], y, bound, f"gemm_lora {what}")
        assert torch.equal(self.y[live:], self.before[live:]), f"{what}: rows of no sequence changed"
