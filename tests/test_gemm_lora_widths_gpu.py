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
