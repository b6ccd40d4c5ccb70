"""What the paged cache's entry points refuse on the host, without a GPU: at the C boundary and for host tensors."""
import ctypes as C

import pytest
import torch


def _lib():
    from rdkv_b200 import _lib
    return _lib.lib()


def _attention(**change):
    a = dict(q=1 << 12, q_tok=1024, q_head=128, dtype=0, T=4, H_q=8, k=1 << 12, k_page=1, k_head=1, k_row=128, v=1 << 12, v_page=1, v_head=1,
             v_row=128, n_pages=2, H_kv=2, page=16, table=1 << 12, stride=4, width=4, q_start=1 << 12, lens=1 << 12, S=1, max_new=4, window=0,
             sinks=0, scale=1.0, out=1 << 12, o_tok=1024, o_head=128, pad=0, rec=None, ws=1 << 12, ws_bytes=1 << 40, stream=None)
    assert set(change) <= set(a)
    return _lib().rdkv_paged_attention(*{**a, **change}.values())


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), 1), (dict(S=-1), 1), (dict(H_q=0), 1), (dict(H_kv=0), 1), (dict(dtype=2), 1), (dict(dtype=7), 1), (dict(window=-1), 1),
    (dict(sinks=-1), 1), (dict(max_new=-1), 1), (dict(width=-1), 1), (dict(n_pages=-1), 1), (dict(H_kv=3), 2), (dict(H_q=34), 2), (dict(page=8), 2),
    (dict(page=24), 2), (dict(page=2048), 2), (dict(q=None), 1), (dict(q_start=None), 1), (dict(lens=None), 1), (dict(table=None), 1),
    (dict(k=None), 1), (dict(v=None), 1), (dict(out=None), 1), (dict(rec=1 << 12), 1), (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float('nan')), 1), (dict(ws=None), 1), (dict(ws=(1 << 12) + 8), 1), (dict(ws_bytes=100), 1),
    (dict(T=0, q=None), 0)])
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
    lib, p = _lib(), 1 << 12
    sec = lambda *n: (C.c_int * len(n))(*n)
    rope = lambda *, dtype=0, T=2, q=p, k=p, pos=p, inv=p, sections=sec(64), axes=1: lib.rdkv_rope_axes(
        q, 512, 128, p, 512, 128, 4, k, 128, 128, p, 128, 128, 1, dtype, T, pos, 2, 0, inv, sections, axes, None)
    assert rope(dtype=3) == 1 and rope(T=-1) == 1 and rope(q=None) == 1 and rope(k=None) == 1 and rope(pos=None) == 1 and rope(inv=None) == 1
    assert rope(sections=None) == 2 and rope(axes=0) == 2 and rope(axes=5) == 2 and rope(sections=sec(63)) == 2
    assert rope(sections=sec(70, -6), axes=2) == 2 and rope(T=0) == 0
    append = lambda *, dtype=0, T=2, H_kv=1, k=p, v=p, kp=p, vp=p, page=16, slots=p, q=p, q_out=p, H_q=4, pos=p, inv=p, sections=sec(64), axes=1: \
        lib.rdkv_paged_append(k, 128, 128, v, 128, 128, H_kv, dtype, T, kp, 2048, 2048, 128, vp, 2048, 2048, 128, 3, page, slots, q, 512, 128,
                              q_out, 512, 128, H_q, pos, 2, 0, inv, sections, axes, None)
    assert append(dtype=-1) == 1 and append(T=-1) == 1 and append(H_kv=0) == 1 and append(k=None) == 1 and append(v=None) == 1
    assert append(kp=None) == 1 and append(vp=None) == 1 and append(page=0) == 1 and append(slots=None) == 1 and append(q=None) == 1
    assert append(q_out=None) == 1 and append(pos=None) == 1 and append(inv=None) == 1 and append(sections=sec(60)) == 2 and append(T=0) == 0


def test_host_tensors_are_refused():
    from rdkv_b200.paged import append_kv, build_block_tables, paged_attention
    from rdkv_b200.rope import rope_axes
    i, x, pages = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 128), torch.zeros(1, 1, 16, 128)
    for call in (lambda: build_block_tables(i, i, i[None], i, 16, 1), lambda: append_kv(x, x, pages, pages, i.long()),
                 lambda: rope_axes(x, x, i, torch.zeros(64)), lambda: paged_attention(x, pages, pages, i[None], torch.zeros(2, dtype=torch.int32), i)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
