"""The paged cache on the GPU: calls at the edge of what its documentation allows."""
import random
from fractions import Fraction

import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF16, F16, INV, check, gen, ints, near, randn, starts

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


# ── starts behind the last row ───────────────────────────────────────────────

def wanted(q, k, v, table, start, lens, T):
    """The reference with the rows' own positions: row t of request i stands at lens[i] - (start[i+1] - t), whether the
    rows up to start[i+1] are all there or not."""
    clamped = [min(max(x, 0), T) for x in start]
    own = [max(0, n - max(0, start[i + 1] - T)) for i, n in enumerate(lens)]
    return R.attention(q, k, v, table, ints(clamped), ints(own))


@pytest.mark.parametrize("max_new", [1, 300])
@pytest.mark.parametrize("start,T", [([0, 0, 300], 203), ([0, 40, 2 ** 31 - 1], 60), ([0, 300, 333], 7), ([-5, 3, 400], 399)])
def test_starts_behind_the_last_row_keep_positions(start, T, max_new):
    """Rows that the tensor does not have are not computed; those it has stand where they stood."""
    from rdkv_b200.paged import paged_attention
    k, v, table = R.build_cache([500, 450], 2, 32, BF16, seed=61)
    q = randn(T, 8, 128, seed=62, dtype=BF16)
    for lens in ([500, 450], [310, 400], [4, 0]):
        got = paged_attention(q, k, v, table, ints(start), ints(lens), max_new=max_new, check_status=True)
        check(got, wanted(q, k, v, table, start, lens, T), f"{lens}")


def test_a_step_with_fewer_token_places_than_tokens():
    """Tables, write and attention of such a step agree on where its rows stand."""
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    kp, vp = (torch.full((9, 2, 16, 128), float("nan"), dtype=BF16, device="cuda") for _ in range(2))     # (what was never written shows)
    plan = build_block_tables(ints([0, 0]), ints([20, 30]), table, ints([5, 6, 7, 8]), 16, 25)
    q, k, v = (randn(25, h, 128, seed=h, dtype=BF16) for h in (8, 2, 2))
    rot = append_kv(k, v, kp, vp, plan.slot_map, q=q, positions=plan.positions, inv_freq=INV())
    got = paged_attention(rot, kp, vp, table, plan.q_start, plan.kv_lens, check_status=True)
    kp, vp = kp.nan_to_num(), vp.nan_to_num()
    check(got, R.attention(rot, kp, vp, table, ints([0, 20, 25]), ints([20, 5])))
