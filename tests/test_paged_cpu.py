"""What the paged cache's entry points refuse on the host, without a GPU: at the C boundary and for host tensors."""
import ctypes as C

import pytest
import torch


def _lib():
    from rdkv_b200 import _lib
    return _lib.lib()


def _attention(**change):
    from rdkv_b200._lib import PagedAttentionArgs
    p = 1 << 12
    fields = dict(q_tok_stride=1024, q_head_stride=128, k_page_stride=1, k_head_stride=1, k_row_stride=128, v_page_stride=1, v_head_stride=1,
                  v_row_stride=128, table_stride=4, dtype=0, n_tokens=4, H_q=8, H_kv=2, n_pages=2, page_size=16, width=4, n_requests=1, max_new=4,
                  window=0, sinks=0, scale=1.0)
    rest = dict(q=p, k=p, v=p, table=p, q_start=p, lens=p, out=p, o_tok=1024, o_head=128, pad=0, rec=None, ws=p, ws_bytes=1 << 40, stream=None)
    assert set(change) <= set(fields) | set(rest)
    args = PagedAttentionArgs(**{n: change.get(n, x) for n, x in fields.items()})
    return _lib().rdkv_paged_attention(C.addressof(args), *(change.get(n, x) for n, x in rest.items()))


@pytest.mark.parametrize("change,status", [
    (dict(n_tokens=-1), 1), (dict(n_requests=-1), 1), (dict(H_q=0), 1), (dict(H_kv=0), 1), (dict(dtype=2), 1), (dict(dtype=7), 1), (dict(window=-1), 1),
    (dict(sinks=-1), 1), (dict(max_new=-1), 1), (dict(width=-1), 1), (dict(n_pages=-1), 1), (dict(H_kv=3), 2), (dict(H_q=34), 2), (dict(page_size=8), 2),
    (dict(page_size=24), 2), (dict(page_size=2048), 2), (dict(q=None), 1), (dict(q_start=None), 1), (dict(lens=None), 1), (dict(table=None), 1),
    (dict(k=None), 1), (dict(v=None), 1), (dict(out=None), 1), (dict(rec=1 << 12), 1), (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float('nan')), 1), (dict(scale=float('inf')), 1), (dict(ws=None), 1), (dict(ws=(1 << 12) + 8), 1), (dict(ws_bytes=100), 1),
    (dict(n_requests=16384, width=1 << 20, page_size=1024), 3), (dict(n_tokens=0, q=None), 0)])
def test_attention_refusals(change, status):
    assert _attention(**change) == status


def test_workspace_refuses_bad_extents():
    f = _lib().rdkv_paged_attention_workspace
    assert f(-1, 1, 8, 2, 1) == -1 and f(1, -1, 8, 2, 1) == -1 and f(1, 1, 0, 2, 1) == -1 and f(1, 1, 8, 0, 1) == -1 and f(1, 1, 8, 2, -1) == -1
    assert f(4, 4, 8, 2, 1) >= 0


def test_tables_refusals():
    f = _lib().rdkv_paged_tables
    p = 1 << 12
    good = [p, p, 2, p, 4, 4, p, 3, None, 16, 5, p, p, p, p, p, p, None]
    for i, bad, status in ((0, None, 1), (1, None, 1), (2, -1, 1), (3, None, 1), (4, 3, 2), (5, -1, 1), (6, None, 1), (7, -1, 1), (9, 0, 1), (10, -1, 1),
                           (11, None, 1), (12, None, 1), (13, None, 1), (14, None, 1), (15, None, 1), (16, None, 1), (2, 16385, 3), (10, 2 ** 31, 3)):
        assert f(*[bad if j == i else x for j, x in enumerate(good)]) == status, i


def test_rotation_and_append_refusals():
    from rdkv_b200._lib import PagedAppendArgs, RopeAxesArgs
    lib, p = _lib(), 1 << 12

    def call(mirror, function, fields, rest, change):
        assert set(change) <= set(fields) | set(rest)
        fields = {n: change.get(n, x) for n, x in fields.items()}
        fields["sections"] = (C.c_int32 * 4)(*fields["sections"])
        args = mirror(**fields)
        return function(C.addressof(args), *(change.get(n, x) for n, x in rest.items()), None)

    def rope(**change):
        return call(RopeAxesArgs, lib.rdkv_rope_axes, dict(H_q=4, H_kv=1, dtype=0, n_tokens=2, n_axes=1, sections=(64,)),
                    dict(q=p, q_out=p, k=p, k_out=p, pos=p, inv=p), change)
    assert rope(dtype=3) == 1 and rope(n_tokens=-1) == 1 and rope(q=None) == 1 and rope(k=None) == 1 and rope(pos=None) == 1 and rope(inv=None) == 1
    assert rope(q_out=None) == 1 and rope(k_out=None) == 1 and rope(n_axes=0) == 2 and rope(n_axes=5) == 2 and rope(sections=(63,)) == 2
    assert rope(sections=(70, -6), n_axes=2) == 2 and rope(n_tokens=0) == 0 and lib.rdkv_rope_axes(None, p, p, p, p, p, p, None) == 1

    def append(**change):
        return call(PagedAppendArgs, lib.rdkv_paged_append,
                    dict(H_q=4, H_kv=1, dtype=0, n_tokens=2, n_pages=3, page_size=16, n_axes=1, sections=(64,)),
                    dict(k=p, v=p, kp=p, vp=p, slots=p, q=p, q_out=p, pos=p, inv=p), change)
    assert append(dtype=-1) == 1 and append(n_tokens=-1) == 1 and append(H_kv=0) == 1 and append(k=None) == 1 and append(v=None) == 1
    assert append(kp=None) == 1 and append(vp=None) == 1 and append(page_size=0) == 1 and append(slots=None) == 1 and append(q=None) == 1
    assert append(q_out=None) == 1 and append(pos=None) == 1 and append(inv=None) == 1 and append(sections=(60,)) == 2 and append(n_tokens=0) == 0
    assert lib.rdkv_paged_append(None, p, p, p, p, p, p, p, p, p, None) == 1


def test_host_tensors_are_refused():
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    from rdkv_b200.rope import rope_axes
    i, x, pages = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 128), torch.zeros(1, 1, 16, 128)
    for call in (lambda: build_block_tables(i, i, i[None], i, 16, 1), lambda: append_kv(x, x, pages, pages, i.long()),
                 lambda: rope_axes(x, x, i, torch.zeros(64)), lambda: paged_attention(x, pages, pages, i[None], torch.zeros(2, dtype=torch.int32), i)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
