"""What the paged cache's entry points refuse on the host: rows that no 16-byte access can take."""
import pytest

from test_paged_cpu import _attention

P = 1 << 12


@pytest.mark.parametrize("change,status", [
    (dict(out=None, rec=P + 4), 1), (dict(out=None, rec=P + 8), 1), (dict(out=P + 2), 1), (dict(q=P + 8), 1), (dict(q=P + 2, max_new=1), 1),
    (dict(q_tok_stride=1023), 2), (dict(q_head_stride=132), 2), (dict(o_tok=1025), 2), (dict(o_head=129), 2)])
def test_attention_refuses_rows_off_16_bytes(change, status):
    assert _attention(**{**dict(k_page_stride=4096, k_head_stride=2048, v_page_stride=4096, v_head_stride=2048, n_pages=0), **change}) == status
