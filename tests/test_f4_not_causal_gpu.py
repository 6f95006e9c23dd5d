"""PagedAttentionF4 without causal masking where a sequence has more tokens than keys: every query sees every key, those in front of
the first key too."""
import pytest

import f4_cases as fc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("csr", [False, True])
@pytest.mark.parametrize("lens", [[(1, 0), (6, 4), (50, 20), (0, 9), (300, 17)], [(8, 5), (2, 0), (5, 1)]], ids=str)
def test_more_tokens_than_keys(session, lens, csr, dim):
    a = fc.Attention(94, lens, dim=dim, csr=csr, causal=False, pad=2)
    a.run(session)
    a.check()
