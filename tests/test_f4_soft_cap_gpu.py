"""PagedAttentionF4's soft cap s -> cap tanh(s / cap) over all positive caps, from those that flatten every score to those that change
none, against 64 bits.

The bound of f4_cases.py holds a capped score to 8 u cap, u = 2^-23, which says nothing where the cap is far above the scores. Here
caps above 128 are held to the score itself. With z = |s| / cap, off by 2 u of it (a product and the constant's rounding):
  * z <= 1/4: s P(z^2), |P - 1| <= 0.021 and the polynomial's own 0.1 u: z's error and the sum's are 0.2 u of P, its last fma and the
    product with s one u each: less than 3 u |s'|, s' the capped score;
  * above: T = 1 - 2 / (1 + e), e = 2^(2 log2(e) z): the exponent is off by 3.5 u of 2 z in units of e, v_exp_f32 and v_rcp_f32 by an
    ulp each, the sum by u: 2 / (1 + e) is off by 2 / (1 + e) (7 z e / (1 + e) + 3) u, at most 3.1 u (at z = 1/4). T is 0.2449 or
    more, so that is 12.7 u of it; the fma, the product with cap and cap's rounding are 2.5 u: less than 16 u |s'|.
Up to 128: 8 u cap, at most 1.3e-4. The rest is as there: e = (d + 4) u scale sum |q_i k_i| of the score in front (a cap never widens
it), then 2 e + 2 |s'| u + u of p."""
import math

import pytest
import torch

import f4_cases as fc
import roost_amd

pytestmark = pytest.mark.gpu

U = fc.U
LENS = [(1, 300), (40, 90), (8, 200), (1, 33)]
TINY = [2.0 ** -149, 1e-42, 2.0 ** -126, 1e-30, 1e-3]
CAPS = [1.0, 30.0, 128.0, 128.5, 1e3, 1e5, 1e8, 2.0 ** 126, 2.5e38, 3.4e38]


def _check(a, cap):
    k_all, v_all = fc.values(*a.cache[:2]), fc.values(*a.cache[2:])
    cap = float(torch.tensor(cap, dtype=torch.float32))
    group, scale, at = a.q_heads // a.kv_heads, a.dim ** -0.5, 0
    for b, (n, keys) in enumerate(a.lens):
        rows, at = slice(at, at + n), at + n
        ids = torch.tensor(a.page_ids[b], dtype=torch.long, device="cuda")
        sees = torch.arange(keys, device="cuda") <= torch.arange(keys - n, keys, device="cuda")[:, None]
        for h in range(a.q_heads):
            k, v = (x[ids, h // group].reshape(-1, a.dim)[:keys] for x in (k_all, v_all))
            q = a.q[rows, h].double()
            s = cap * torch.tanh((q @ k.T) * scale / cap)
            e = (a.dim + 4) * U * scale * (q.abs() @ k.abs().T) + (8 * U * cap if cap <= 128 else 16 * U * s.abs()) + 2.0 ** -126
            s = s.masked_fill(~sees, -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None])
            want = p @ v
            err = ((2 * (e + 2 * s.abs() * U).masked_fill(~sees, 0.0).amax(1) + U) + keys * U)[:, None]
            assert (err < 0.5).all()
            bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -7) * (2.0 ** -8 + 2 * err) * (p @ v.abs()) + \
                2.0 ** -126 * (sees.double() @ v.abs()) + 2.0 ** -133
            fc._within(a.out[rows, h], want, bound, f"cap {cap} sequence {b} head {h} out")
            near = err[:, 0] * math.log2(math.e) + 4 * U * (lse / math.log(2)).abs()
            fc._within(a.lse[rows, h], lse / math.log(2), near, f"cap {cap} sequence {b} head {h} lse")


@pytest.mark.parametrize("std", [1.0, 40.0])
@pytest.mark.parametrize("cap", CAPS, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads", [8, 20])
def test_caps(session, q_heads, dim, cap, std):
    a = fc.Attention(90, LENS, q_heads=q_heads, kv_heads=2 if q_heads == 8 else 1, dim=dim, soft_cap=cap, std=std)
    a.run(session)
    _check(a, cap)


@pytest.mark.parametrize("cap", TINY, ids=str)
def test_caps_that_flatten_every_score(session, cap):
    a = fc.Attention(91, LENS, dim=128, soft_cap=cap)
    a.q[0, 0] = 0  # scores of exactly 0
    a.run(session)
    _check(a, cap)
