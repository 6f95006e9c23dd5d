"""A transformer layer of a worker step as a user runs it, with an adapter for each sequence: AddRmsNorm, the q/k/v projection
(GemmLora), QkNorm + Rope + CacheWrite, PagedAttention, the output projection onto the residual (GemmLora), AddRmsNormQuant, the
gate/up projection of 8-bit rows (GemmLora), SiluMulQuant and the down projection of 8-bit rows onto the residual (GemmLora).

Every call is checked against its definition in 64 bits on the inputs that it had on the GPU, with the bounds of fused_cases.py;
the attention, which has tests of its own, against a float32 definition within 2e-2. The layer runs eagerly and then as one
captured graph over the same buffers, with the same results bit for bit at every replay."""
import pytest
import torch

import fused_cases as fc
import roost_amd
from fused_cases import BF16, F8, F32, Lora

pytestmark = pytest.mark.gpu

HQ, HK, HD, PAGE, EPS, THETA = 8, 2, 128, 16, 1e-6, 1e6
DIM, MLP = HQ * HD, 2816


class Pool:
    """A projection's weight and its adapters, of pool rank 16."""

    def __init__(self, v, in_dim, out_dim, adapters, x=BF16):
        w = v(out_dim, in_dim, std=in_dim ** -0.5)
        self.w_scale = None
        if x == F8:
            self.w_scale = w.abs().amax(1) / 448
            w = w / self.w_scale[:, None]
        self.w = w.to(x)
        self.a = v(adapters, 16, in_dim, std=in_dim ** -0.5).to(BF16)
        self.b = v(adapters, out_dim, 16, std=0.25).to(BF16)
        self.scale = 0.5 + v(adapters, std=0.1).abs()


class Layer:
    def __init__(self, session, lens, kv_lens, slots, pad):
        g = torch.Generator(device="cuda").manual_seed(sum(lens))
        v = lambda *s, std=1.0: torch.randn(s, generator=g, device="cuda") * std  # noqa: E731
        i32 = lambda a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
        self.session, self.lens, self.kv_lens, self.slots = session, lens, kv_lens, slots
        self.live, self.t = sum(lens), sum(lens) + pad
        t, adapters = self.t, 5
        self.ranks_h = [16, 8, 3, 0, 13]
        self.ranks = i32(self.ranks_h).cuda()
        self.slots_d, self.cu = i32(slots).cuda(), i32([sum(lens[:i]) for i in range(len(lens) + 1)]).cuda()
        self.x, self.residual0 = v(t, DIM).to(BF16), v(t, DIM, std=2.0).to(BF16)
        self.norm1, self.norm2 = ((1 + v(DIM, std=0.1)).to(BF16) for _ in range(2))
        self.q_norm, self.k_norm = ((1 + v(HD, std=0.1)).to(BF16) for _ in range(2))
        self.qkv, self.out = Pool(v, DIM, (HQ + 2 * HK) * HD, adapters), Pool(v, DIM, DIM, adapters)
        self.up, self.down = Pool(v, DIM, 2 * MLP, adapters, F8), Pool(v, MLP, DIM, adapters, F8)
        # Pages in any order, the histories in them.
        pages = [-(-n // PAGE) for n in kv_lens]
        perm = torch.randperm(sum(pages) + 3, generator=torch.Generator().manual_seed(1)).int()
        self.indptr_h = i32([sum(pages[:i]) for i in range(len(pages) + 1)])
        self.last_h = i32([(n - 1) % PAGE + 1 for n in kv_lens])
        self.q_indptr_h = self.cu.cpu()
        self.indptr, self.last, self.indices = self.indptr_h.cuda(), self.last_h.cuda(), perm[:sum(pages)].cuda()
        shape = (sum(pages) + 3, PAGE, HK, HD)
        self.k_cache, self.v_cache = v(*shape).to(BF16), v(*shape).to(BF16)
        positions, mapping = [], []
        for s, (n, kv) in enumerate(zip(lens, kv_lens)):
            for p in range(kv - n, kv):
                positions.append(p)
                mapping.append(int(perm[self.indptr_h[s] + p // PAGE]) * PAGE + p % PAGE)
        self.positions, self.mapping = i32(positions + [0] * pad).cuda(), torch.tensor(mapping + [-1] * pad).cuda()
        e = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        self.residual, self.h = self.residual0.clone(), e(t, DIM)
        self.h8, self.h8_scale = e(t, DIM, dtype=F8), e(t, 1, dtype=F32)
        self.qkv_y, self.q, self.attn = e(t, (HQ + 2 * HK) * HD), e(t, HQ, HD), e(t, HQ, HD)
        self.gate_up, self.act8, self.act8_scale = e(t, 2 * MLP), e(t, MLP, dtype=F8), e(t, 1, dtype=F32)

    def lora(self, key, pool, x, y, x_scale=None, addend=None):
        p = roost_amd.gemm_lora_params(x, pool.w, pool.a, pool.b, pool.scale, self.slots_d, self.cu, y, ranks=self.ranks,
                                       x_scale=x_scale, w_scale=pool.w_scale, addend=addend)
        roost_amd.gemm_lora(self.session, p, key=key)

    def check_lora(self, what, pool, x, y, x_scale=None, addend=None):
        c = Lora.__new__(Lora)
        c.lens, c.slots, c.x, c.y, c.before, c.addend = self.lens, self.slots, x, y, y, addend
        c.weight, c.x_scale, c.w_scale, c.low = pool.w, x_scale, pool.w_scale, BF16
        c.lora_a, c.lora_b, c.lora_scale = pool.a, pool.b, pool.scale
        c.adapters, c.max_rank, c.ranks_h = 5, 16, self.ranks_h
        c.check(what)

    def run(self, check=False):
        s, kept = self.session, None

        def looked(f, *args, **kw):
            if check:
                torch.cuda.synchronize()
                f(*args, **kw)

        # h = norm(residual + x), the residual in place
        p = roost_amd.add_rms_norm_params(self.x, self.residual, self.norm1, self.residual, self.h, eps=EPS)
        roost_amd.add_rms_norm(s, p)
        looked(self.check_norm, self.x, self.residual0)
        self.lora("qkv", self.qkv, self.h, self.qkv_y)
        looked(self.check_lora, "q/k/v", self.qkv, self.h, self.qkv_y)
        roost_amd.qkv_qk_norm_rope_cache_write(s, self.qkv_y, self.q, self.q_norm, self.k_norm, self.positions, self.k_cache,
                                               self.v_cache, self.mapping, tokens=self.t, q_heads=HQ, kv_heads=HK,
                                               head_dim=HD, page_size=PAGE, eps=EPS, theta=THETA)
        s.run(s.lib.entry(roost_amd.ATTENTION_VARIANT), self.attention, self.attention_ws)
        looked(self.check_attention)
        attn = self.attn.view(self.t, DIM)
        kept = self.residual.clone() if check else None
        self.lora("out", self.out, attn, self.residual, addend=self.residual)  # onto the residual, in place
        looked(self.check_lora, "output", self.out, attn, self.residual, addend=kept)
        roost_amd.add_rms_norm_quant(s, roost_amd.add_rms_norm_quant_params(self.residual, None, self.norm2, None, self.h8,
                                                                            self.h8_scale, eps=EPS))
        looked(self.check_norm_quant)
        self.lora("up", self.up, self.h8, self.gate_up, x_scale=self.h8_scale.view(-1))
        looked(self.check_lora, "gate/up", self.up, self.h8, self.gate_up, x_scale=self.h8_scale.view(-1))
        roost_amd.silu_mul_quant(s, roost_amd.silu_mul_quant_params(self.gate_up[:, :MLP], self.gate_up[:, MLP:], self.act8,
                                                                    self.act8_scale))
        looked(self.check_silu)
        kept = self.residual.clone() if check else None
        self.lora("down", self.down, self.act8, self.residual, x_scale=self.act8_scale.view(-1), addend=self.residual)
        looked(self.check_lora, "down", self.down, self.act8, self.residual, x_scale=self.act8_scale.view(-1), addend=kept)

    def check_norm(self, x, residual):
        _, want = fc.norm64(x, residual, self.norm1, EPS)
        fc.assert_within(self.h, want, fc.rounded_bound(want, BF16, fc.NORM * want.abs()), "norm")
        assert torch.equal(self.residual, (x.float() + residual.float()).to(BF16))

    def check_norm_quant(self):
        _, want = fc.norm64(self.residual, None, self.norm2, EPS)
        fc.assert_quantised(self.h8, self.h8_scale, want, 0, fc.NORM, "norm in 8 bits")

    def check_silu(self):
        live = self.gate_up[:self.live]
        want = fc.silu64(live[:, :MLP], live[:, MLP:])
        fc.assert_quantised(self.act8[:self.live], self.act8_scale[:self.live], want, 0, fc.SILU, "activation in 8 bits")

    def check_attention(self):
        at = 0
        for s, (n, kv) in enumerate(zip(self.lens, self.kv_lens)):
            pages = self.indices[self.indptr_h[s]:self.indptr_h[s + 1]].long()
            k, v = (c[pages].reshape(-1, HK, HD)[:kv].float().repeat_interleave(HQ // HK, 1)
                    for c in (self.k_cache, self.v_cache))
            q = self.q[at:at + n].float()
            score = (q[:, None] * k[None]).sum(-1) * HD ** -0.5  # [n, kv, heads]
            past = torch.arange(kv, device="cuda")[None] <= torch.arange(kv - n, kv, device="cuda")[:, None]
            p = torch.softmax(score.masked_fill(~past[..., None], float("-inf")), 1)
            want = (p[..., None] * v[None]).sum(1)
            off = (self.attn[at:at + n].float() - want).abs().max()
            assert off < 2e-2, f"attention of sequence {s} off by {float(off)}"
            at += n

    def plan(self):
        self.attention = roost_amd.paged_attention_params(
            self.q[:self.live], self.attn[:self.live], self.k_cache, self.v_cache, self.q_indptr, self.indptr, self.indices,
            self.last, q_indptr_host=self.q_indptr_h, kv_indptr_host=self.indptr_h, kv_last_page_len_host=self.last_h,
            batch=len(self.lens), q_heads=HQ, kv_heads=HK, head_dim=HD, page_size=PAGE)
        entry = self.session.lib.entry(roost_amd.ATTENTION_VARIANT)
        self.attention_ws = self.session.prepare(entry, self.attention, key="step")

    @property
    def q_indptr(self):
        return self.cu


@pytest.mark.parametrize("lens,kv_lens,slots,pad", [
    ([1], [37], [2], 0),                                                  # one chat
    ([1] * 13, [3, 40, 1, 77, 16, 100, 5, 33, 64, 2, 90, 17, 48], [i % 6 - 1 for i in range(13)], 3),  # a decode bucket
    ([1, 1, 70, 1, 33], [50, 9, 70, 128, 90], [0, 4, 1, -1, 2], 0),       # decode rows and prompt chunks
    ([300], [300], [3], 0),                                               # a prompt; its adapter has rank 0
])
def test_layer(session, lens, kv_lens, slots, pad):
    stream = torch.cuda.Stream()
    s = roost_amd.OpSession(session.lib, device=0, stream=stream)
    with torch.cuda.stream(stream):
        layer = Layer(s, lens, kv_lens, slots, pad)
        layer.plan()
        layer.run(check=True)
        torch.cuda.synchronize()
        live, want = layer.live, layer.residual.clone()
        k, v = layer.k_cache.clone(), layer.v_cache.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        layer.run()
    for _ in range(3):
        with torch.cuda.stream(stream):
            layer.residual.copy_(layer.residual0)
            layer.gate_up.fill_(7)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(layer.residual[:live], want[:live])
            assert torch.equal(layer.k_cache, k) and torch.equal(layer.v_cache, v)
    s.close()
