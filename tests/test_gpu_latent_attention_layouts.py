"""
The latent-attention operators in layouts beside the usual ones.
"""
import pytest
import torch

from test_gpu_latent_attention import BF, _check_paged, _paged_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[90, 31, 64], [5, 8, 1]])
def test_block_tables_in_other_layouts(lens):
    """Columns first, and a slice of a wider table; the one-page tables' columns have any stride."""
    from lazylora_b200.core import latent_attention as A
    q, cache, bt, sl, rows = _paged_case(BF, lens, 1, 4, 128, 64, 8, 13)
    bt = bt[:, :(max(lens) + 7) // 8]
    want = A.paged_latent_attention(q, cache, bt.contiguous(), sl, 128, 0.1)
    _check_paged(*want, q, rows, 128, 0.1)
    for other in (bt, bt.t().contiguous().t(), torch.cat([bt, bt], 1)[:, bt.shape[1]:], bt.repeat_interleave(2, 1)[:, ::2]):
        got = A.paged_latent_attention(q, cache, other, sl, 128, 0.1)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    A.check_status()
