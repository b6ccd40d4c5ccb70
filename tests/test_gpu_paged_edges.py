"""The paged cache on the GPU: calls at the edge of what its documentation allows."""
import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF16, F16, INV, check, gen, ints, randn, starts

pytestmark = pytest.mark.gpu


def test_records_off_16_bytes_are_refused():
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([64], 2, 16, F16, seed=1)
    q = randn(1, 8, 128, seed=2, dtype=F16)
    flat = torch.zeros(8 * 132 + 4, device="cuda")
    for shift in (1, 2, 3):
        with pytest.raises(ValueError, match="16 bytes"):
            paged_attention(q, k, v, table, ints([0, 1]), ints([64]), out_partial=flat[shift:shift + 8 * 132].view(8, 132))
    paged_attention(q, k, v, table, ints([0, 1]), ints([64]), out_partial=flat[4:].view(8, 132))
    assert (flat[:4] == 0).all() and (flat[5::132] > 0).all()
