"""What the paged cache's entry points refuse on the host: rows that no 16-byte access can take, limits that are none."""
import ctypes as C

import pytest

from test_paged_cpu import _attention

P = 1 << 12


@pytest.mark.parametrize("change,status", [
    (dict(out=None, rec=P + 4), 1), (dict(out=None, rec=P + 8), 1), (dict(out=P + 2), 1), (dict(q=P + 8), 1), (dict(q=P + 2, max_new=1), 1),
    (dict(q_tok_stride=1023), 2), (dict(q_head_stride=132), 2), (dict(o_tok=1025), 2), (dict(o_head=129), 2)])
def test_attention_refuses_rows_off_16_bytes(change, status):
    assert _attention(**{**dict(k_page_stride=4096, k_head_stride=2048, v_page_stride=4096, v_head_stride=2048, n_pages=0), **change}) == status


@pytest.mark.parametrize("wait_us,status", [(-1, 1), (4000001, 1), (0, 0), (4000000, 0)])
def test_limits_of_waits(wait_us, status):
    from rdkv_b200._lib import PagedAttentionArgs, lib
    args = PagedAttentionArgs(H_q=8, H_kv=2, page_size=16, scale=1.0)     # (no tokens: nothing is launched)
    assert lib().rdkv_paged_attention_within(C.addressof(args), *[None] * 7, 0, 0, 0, None, None, 0, wait_us, None) == status
