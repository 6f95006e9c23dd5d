"""GemmLora over inner lengths that end inside a step of 128 bytes, long enough for every ring of steps to come round, against
its definition in 64 bits; the bounds are derived in fused_cases.py."""
import pytest
import torch

import roost_amd
from fused_cases import BF16, F8, F32, Lora

pytestmark = pytest.mark.gpu


def _run(session, c):
    c.y.copy_(c.before)
    roost_amd.gemm_lora(session, c.params())
    torch.cuda.synchronize()


# Rows of 8 bits, whose adapters' rows are twice as long: the last step's second half is whole, cut, or past the rows' end
# (in_dim % 128 of 16 to 64). One launch; low-rank rows by 16 (ranks in blocks of 16 and of 32) and by 64 rows.
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("in_dim", [528, 576, 1040, 1088, 1136, 2112, 2880, 4160])
@pytest.mark.parametrize("lens,max_rank", [([1], 16), ([3, 5], 8), ([1] * 40, 16), ([1] * 300, 32), ([2] * 40, 128),
                                           ([3001, 1, 3200], 16), ([3001, 1, 3200], 32), ([3001, 1, 3200], 128)])
def test_low_rank_rows_of_8_bit_rows(session, lens, max_rank, in_dim, out):
    for shared in (True, False):
        c = Lora(in_dim + max_rank, lens, [(5 * i + 1) % 4 for i in range(len(lens))], in_dim=in_dim, out_dim=72,
                 max_rank=max_rank, ranks=[max_rank, max_rank, max_rank - 3, max_rank - 1], x=F8, out=out, shared=shared)
        _run(session, c)
        c.check(f"{len(lens)} sequences, inner length {in_dim}, shared {shared}")
        first = c.y.clone()
        for _ in range(2):
            _run(session, c)
            assert torch.equal(c.y, first)


def _lens(tokens, long):
    """Sequences of one token to `long`, and empty ones."""
    lens, left, k = [], tokens, 0
    while left:
        lens.append(min(left, [1, long, 0, 5, long // 2, 30][k % 6]))
        left -= lens[-1]
        k += 1
    return lens


# Rows x outputs that take each of the tilings, with as many steps of 128 bytes as make its ring of stages come round twice and
# more (by tiles: 2 to 4 stages; by wavefronts that split the steps: 4 or 8 of them and 2 to 4 stages each), the last of them
# whole or cut. With a few adapters in each tile, whose steps follow in the same ring.
@pytest.mark.parametrize("x,out", [(BF16, BF16), (BF16, F32), (F32, F32), (F8, BF16), (F8, F32)])
@pytest.mark.parametrize("cut", [0, 16, 48, 80, 112])
@pytest.mark.parametrize("tokens,out_dim,steps", [
    (5, 300, 41),      # one launch
    (13, 2100, 41),    # 16 outputs x 16 rows
    (13, 5001, 41),    # 32 x 16
    (31, 2100, 41),    # 16 x 32
    (31, 5001, 41),    # 32 x 32
    (63, 6100, 41),    # 32 x 64
    (300, 2100, 41),   # 80 x 64
    (300, 5001, 10),   # 64 x 64
    (1020, 2100, 10),  # 128 x 128
    (1500, 2901, 10),  # 256 x 128
    (2601, 4200, 10),  # 256 x 256
    (4201, 4200, 10),  # 256 x 256 and 128 x 128
])
def test_rings_come_round(session, tokens, out_dim, steps, cut, x, out):
    size = torch.tensor([], dtype=x).element_size()
    lens = [tokens] if tokens == 5 else _lens(tokens, 70)
    c = Lora(steps + cut + tokens, lens, [(3 * i + 1) % 4 for i in range(len(lens))], in_dim=(128 * steps + cut) // size,
             out_dim=out_dim, max_rank=16, ranks=[16, 9, 3, 16], x=x, out=out, pad=1)
    _run(session, c)
    c.check(f"{tokens} x {out_dim}, {128 * steps + cut} bytes")
    first = c.y.clone()
    _run(session, c)
    assert torch.equal(c.y, first)
