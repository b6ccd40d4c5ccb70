"""The paged cache: uncompressed keys and values of running requests, before (or beside) their packed form.

Keys and values live in pages of ``page_size`` tokens, ``k_pages`` / ``v_pages`` ``[n_pages,H_kv,page_size,128]``
(any strides whose rows are contiguous), and a request owns the pages its row of ``block_tables`` lists.  A step of a
batch whose requests have ``ctx_lens`` tokens in the cache and ``new_lens`` new ones is

    plan = build_block_tables(ctx_lens, new_lens, block_tables, free_pages, page_size, n_tokens)   # once
    q = append_kv(k, v, k_pages, v_pages, plan.slot_map, q=q, positions=plan.positions,            # in every layer
                  inv_freq=inv_freq)
    out = paged_attention(q, k_pages, v_pages, block_tables, plan.q_start, plan.kv_lens, max_new=...)

for chunks of a prompt, single decoded tokens and both at once.  All lengths are read on the device: nothing
here waits for the GPU, and a captured step can be replayed with other lengths.  The pages of a prompt that is complete
are what :mod:`rdkv_b200.packing` compresses, and :func:`paged_attention` can leave records that
:func:`rdkv_b200.decode.lse_combine` merges with those of packed layers.

Every call launches on the current stream of its tensors' device.  A call's scratch memory is its own (allocated by
the call), so calls on different streams and captured graphs do not share any.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Sequence

import torch
from torch import Tensor

from ._lib import (HEAD_DIM, PARTIAL_STRIDE, CallCache, PagedAppendArgs, PagedAttentionArgs, apart, check, extent, fits_32_bits, footprint, lib,
                   q_dtype_tag, raw_stream, require_cuda, separate_rows, share_memory)
from .rope import axes_check, empty_rows, plain_sections

MAX_REQUESTS = 16384
_TABLES_CALLS, _APPEND_CALLS, _ATTENTION_CALLS = CallCache(), CallCache(), CallCache()


class PagedPlan(NamedTuple):
    """What :func:`build_block_tables` worked out for a step."""
    slot_map: Tensor      # int64 [n_tokens]  slot (page * page_size + row) of every new token, -1: none
    positions: Tensor     # int32 [n_tokens]  its position in its request (padding: 0)
    q_start: Tensor       # int32 [S+1]       first new token of every request
    kv_lens: Tensor       # int32 [S]         tokens of every request, the new ones included
    free_next: Tensor     # int32 [1]         first entry of the free list that is still free
    missing: Tensor       # int32 [1]         pages that could not be had


def _int32(t: Tensor, name: str, dim: int) -> None:
    require_cuda(t, name)
    if t.dtype != torch.int32 or t.dim() != dim or (t.dim() > 0 and t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be an int32 tensor of {dim} dimension(s) with contiguous rows")


def _same_device(dev, **tensors: Optional[Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} must live on {dev}, got {t.device}")


def _check_plan_apart(out: "PagedPlan", **read: Optional[Tensor]) -> None:
    """Refuses a plan whose tensors share memory with one another or with the arguments that the launch reads."""
    places = [(n, t, t.data_ptr(), t.data_ptr() + extent(t)) for n, t in {**out._asdict(), **read}.items() if t is not None and t.numel() > 0]
    mine = [x for x in places if x[0] not in read]
    for i, (name, t, begin, end) in enumerate(mine):
        for other, x, b, e in places[i + 1:]:
            if begin < e and b < end and share_memory(t, x):
                why = "which other blocks of the launch still read" if other in read else "which is written too"
                raise ValueError(f"out.{name} shares memory with {other}, {why}")


def build_block_tables(ctx_lens: Tensor, new_lens: Tensor, block_tables: Tensor, free_pages: Tensor, page_size: int, n_tokens: int,
                       *, free_start: Optional[Tensor] = None, out: Optional[PagedPlan] = None) -> PagedPlan:
    """Gives the requests of a step the pages they lack and every new token its slot; one launch.

    ctx_lens, new_lens int32 [S] (S up to 16384; negative counts as zero): tokens in the cache, new tokens.
    block_tables int32 [S,width]: the pages a request holds (``ceil(ctx/page_size)`` entries) are read, those of its new
    pages are written IN PLACE, everything behind them is left as it was.  free_pages int32 [F]: page numbers to hand
    out, in request order, from entry ``free_start`` (int32 [1], default 0) on; the caller goes on at ``free_next`` (a
    tensor of its own: ``free_start`` is not changed).  n_tokens: length of the step's token buffers; tokens behind
    the last request's are padding (slot -1, position 0).

    A page that is not to be had (the free list is used up: entry -1; the table is too narrow: no entry) leaves its
    tokens without a slot (-1): :func:`append_kv` does not write them and :func:`paged_attention` does not see them.
    ``missing`` counts such pages.  ``out``: a plan of the same S and n_tokens to write into; its tensors must not share memory with one
    another or with the arguments (a step's ``kv_lens`` are the next one's ``ctx_lens``: take two plans in turn, or copy)."""
    n_tokens, page_size = int(n_tokens), int(page_size)
    key = (ctx_lens.shape, ctx_lens.stride(), ctx_lens.dtype, ctx_lens.get_device(), new_lens.shape, new_lens.stride(), new_lens.dtype,
           new_lens.get_device(), block_tables.shape, block_tables.stride(), block_tables.dtype, block_tables.get_device(), free_pages.shape,
           free_pages.stride(), free_pages.dtype, free_pages.get_device(), page_size, n_tokens,
           None if free_start is None else (free_start.shape, free_start.dtype, free_start.get_device()))
    call = _TABLES_CALLS.get(key)
    if call is None:
        _int32(ctx_lens, "ctx_lens", 1); _int32(new_lens, "new_lens", 1); _int32(block_tables, "block_tables", 2)
        _int32(free_pages, "free_pages", 1)
        S, dev = ctx_lens.shape[0], ctx_lens.device
        if new_lens.shape[0] != S or block_tables.shape[0] != S:
            raise ValueError(f"new_lens and block_tables must have {S} rows, got {new_lens.shape[0]} and {block_tables.shape[0]}")
        if S > MAX_REQUESTS:
            raise ValueError(f"{S} requests: at most {MAX_REQUESTS}")
        if page_size < 1 or n_tokens < 0:
            raise ValueError(f"bad page_size {page_size} or n_tokens {n_tokens}")
        fits_32_bits(page_size=page_size, n_tokens=n_tokens, width=block_tables.shape[1], free_pages=free_pages.shape[0])
        if S > 1 and block_tables.shape[1] > 0 and block_tables.stride(0) < block_tables.shape[1]:
            raise ValueError("rows of block_tables overlap")
        if free_start is not None:
            _int32(free_start, "free_start", 1)
            if free_start.shape[0] != 1:
                raise ValueError("free_start must have one element")
        _same_device(dev, new_lens=new_lens, block_tables=block_tables, free_pages=free_pages, free_start=free_start)
        call = _TABLES_CALLS.remember(key, (S, (block_tables.stride(0), block_tables.shape[1]), free_pages.shape[0], dev.index))
    S, table, n_free, index = call
    if out is None:
        ints = ctx_lens.new_empty(n_tokens + 2 * S + 3)
        out = PagedPlan(ctx_lens.new_empty(n_tokens, dtype=torch.int64), *ints.unsafe_split_with_sizes((n_tokens, S + 1, S, 1, 1)))
    else:
        for name, n in (("positions", n_tokens), ("q_start", S + 1), ("kv_lens", S), ("free_next", 1), ("missing", 1)):
            t = getattr(out, name)
            _int32(t, f"out.{name}", 1)
            if t.shape[0] != n:
                raise ValueError(f"out.{name} must have {n} elements")
        if out.slot_map.dtype != torch.int64 or tuple(out.slot_map.shape) != (n_tokens,) or not out.slot_map.is_contiguous():
            raise ValueError(f"out.slot_map must be a contiguous int64 tensor of {n_tokens} elements")
        _same_device(ctx_lens.device, **{f"out.{n}": t for n, t in out._asdict().items()})
        _check_plan_apart(out, ctx_lens=ctx_lens, new_lens=new_lens, free_pages=free_pages, free_start=free_start, block_tables=block_tables)
    slot_map, positions, q_start, kv_lens, free_next, missing = out
    status = lib().rdkv_paged_tables(
        ctx_lens.data_ptr(), new_lens.data_ptr(), S, block_tables.data_ptr(), *table, free_pages.data_ptr(), n_free,
        None if free_start is None else free_start.data_ptr(), page_size, n_tokens, slot_map.data_ptr(), positions.data_ptr(),
        q_start.data_ptr(), kv_lens.data_ptr(), free_next.data_ptr(), missing.data_ptr(), raw_stream(index))
    if status:
        check(status, "rdkv_paged_tables")
    return out


def _check_pages(k_pages: Tensor, v_pages: Tensor, written: bool) -> None:
    require_cuda(k_pages, "k_pages"); require_cuda(v_pages, "v_pages")
    if k_pages.dim() != 4 or k_pages.shape[3] != HEAD_DIM or k_pages.shape != v_pages.shape:
        raise ValueError(f"k_pages and v_pages must be [n_pages,H_kv,page_size,{HEAD_DIM}], got {tuple(k_pages.shape)} and "
                         f"{tuple(v_pages.shape)}")
    if k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must have one dtype")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError("rows of k_pages and v_pages must be contiguous")
    separate_rows(k_pages, "k_pages", written); separate_rows(v_pages, "v_pages", written)


def append_kv(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, slot_map: Tensor, *, q: Optional[Tensor] = None,
              positions: Optional[Tensor] = None, inv_freq: Optional[Tensor] = None, sections: Optional[Sequence[int]] = None,
              q_out: Optional[Tensor] = None) -> Optional[Tensor]:
    """Writes the new tokens' keys and values to their slots; with ``positions`` the keys, and the queries
    ``q``, are rotated on the way (as :func:`rdkv_b200.rope.rope_axes` does).  One launch.

    k, v [T,H_kv,128]; k_pages, v_pages [n_pages,H_kv,page_size,128] of the same dtype (fp16 / bf16 / fp32); slot_map int64
    [T]: slot of every token; a slot below zero or behind the last page is not written.  The slots of a call must
    differ from one another.  q [T,H_q,128] of the same dtype goes to ``q_out`` (default: a new tensor; may be q
    itself, but share no other memory with q, k or v), which is returned; k is not changed.  k and v may be rows of pages that the
    call does not write to.  positions [T] or [axes,T], inv_freq and sections: see ``rope_axes``."""
    if sections is not None:
        sections = plain_sections(sections)
    key = (k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype, v.get_device(), k_pages.shape, k_pages.stride(),
           k_pages.dtype, k_pages.get_device(), v_pages.shape, v_pages.stride(), v_pages.dtype, v_pages.get_device(), slot_map.shape,
           slot_map.stride(), slot_map.dtype, slot_map.get_device(), sections,
           None if positions is None else (positions.shape, positions.stride(), positions.dtype, positions.get_device()),
           None if inv_freq is None else (inv_freq.shape, inv_freq.stride(), inv_freq.dtype, inv_freq.get_device()),
           None if q is None else (q.shape, q.stride(), q.dtype, q.get_device()),
           None if q_out is None else (q_out.shape, q_out.stride(), q_out.dtype, q_out.get_device()))
    call = _APPEND_CALLS.get(key)
    if call is None:
        call = _APPEND_CALLS.remember(key, _append_check(k, v, k_pages, v_pages, slot_map, q, positions, inv_freq, sections, q_out))
    args, _, index, dense, marks = call
    k_ptr, v_ptr, kp_ptr, vp_ptr = k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    if kp_ptr == vp_ptr and kp_ptr != 0:
        raise ValueError("k_pages and v_pages must not share memory")
    if marks is not None:
        q_mark, qo_mark, k_mark, v_mark, q_like = marks
        q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
        if not ((q_like and q_ptr == qo_ptr or apart(q_out, qo_ptr, qo_mark, q, q_ptr, q_mark)) and apart(q_out, qo_ptr, qo_mark, k, k_ptr, k_mark)
                and apart(q_out, qo_ptr, qo_mark, v, v_ptr, v_mark)):
            raise ValueError("q_out may be q itself, but must share no other memory with q, k or v")
    elif q is not None:
        q_out = empty_rows(q, dense)
    status = lib().rdkv_paged_append(
        args, k_ptr, v_ptr, kp_ptr, vp_ptr, slot_map.data_ptr(), None if q is None else q.data_ptr(),
        None if q is None else q_out.data_ptr(), None if positions is None else positions.data_ptr(),
        None if positions is None else inv_freq.data_ptr(), raw_stream(index))
    if status:
        check(status, "rdkv_paged_append")
    return q_out


def _append_check(k, v, k_pages, v_pages, slot_map, q, positions, inv_freq, sections, q_out):
    require_cuda(k, "k"); require_cuda(v, "v"); require_cuda(slot_map, "slot_map")
    _check_pages(k_pages, v_pages, True)
    n_pages, H_kv, page_size, _ = k_pages.shape
    if k.dim() != 3 or tuple(k.shape[1:]) != (H_kv, HEAD_DIM) or v.shape != k.shape:
        raise ValueError(f"k and v must be [T,{H_kv},{HEAD_DIM}], got {tuple(k.shape)} and {tuple(v.shape)}")
    T, dev = k.shape[0], k.device
    fits_32_bits(T=T, n_pages=n_pages, page_size=page_size, H_q=0 if q is None else q.numel() // max(T * HEAD_DIM, 1))
    if k.dtype != k_pages.dtype or v.dtype != k_pages.dtype:
        raise ValueError(f"k and v must have the pages' dtype {k_pages.dtype}")
    if k.stride(2) != 1 or v.stride(2) != 1:
        raise ValueError("rows of k and v must be contiguous")
    if slot_map.dtype != torch.int64 or tuple(slot_map.shape) != (T,) or (T > 1 and slot_map.stride(0) != 1):
        raise ValueError(f"slot_map must be a contiguous int64 tensor of {T} elements")
    tag = q_dtype_tag(k)
    if (positions is None) != (inv_freq is None) or (positions is None and (q is not None or sections is not None)):
        raise ValueError("q and sections need positions and inv_freq; positions needs inv_freq")
    axes = {} if positions is None else axes_check(positions, inv_freq, sections, T, dev)
    qs, qos, H_q = (0, 0), (0, 0), 0
    if q is None:
        if q_out is not None:
            raise ValueError("q_out needs q")
    else:
        require_cuda(q, "q")
        if q.dim() != 3 or q.shape[0] != T or q.shape[2] != HEAD_DIM or q.dtype != k.dtype or q.stride(2) != 1:
            raise ValueError(f"q must be [{T},H_q,{HEAD_DIM}] {k.dtype} with contiguous rows, got {tuple(q.shape)} {q.dtype}")
        if q_out is not None and (q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.stride(2) != 1):
            raise ValueError("q_out must have q's shape and dtype and contiguous rows")
        if q_out is not None:
            separate_rows(q_out, "q_out")
        H_q = q.shape[1]
        qs, qos = q.stride(), (H_q * HEAD_DIM, HEAD_DIM) if q_out is None else q_out.stride()
    _same_device(dev, v=v, k_pages=k_pages, v_pages=v_pages, slot_map=slot_map, q=q, q_out=q_out)
    ks, vs, kp, vp = k.stride(), v.stride(), k_pages.stride(), v_pages.stride()
    args = PagedAppendArgs(
        k_tok_stride=ks[0], k_head_stride=ks[1], v_tok_stride=vs[0], v_head_stride=vs[1], k_page_stride=kp[0], k_page_head_stride=kp[1],
        k_page_row_stride=kp[2], v_page_stride=vp[0], v_page_head_stride=vp[1], v_page_row_stride=vp[2], q_tok_stride=qs[0],
        q_head_stride=qs[1], q_out_tok_stride=qos[0], q_out_head_stride=qos[1], H_q=H_q, H_kv=H_kv, dtype=tag, n_tokens=T, n_pages=n_pages,
        page_size=page_size, **axes)
    marks = None if q_out is None else (footprint(q), footprint(q_out), footprint(k), footprint(v), q_out.stride() == q.stride())
    return C.addressof(args), args, dev.index, q is not None and q.is_contiguous(), marks


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_tables: Tensor, q_start: Tensor, kv_lens: Tensor, *,
                    max_new: Optional[int] = None, window: int = 0, sinks: int = 0, scale: Optional[float] = None,
                    out: Optional[Tensor] = None, out_partial: Optional[Tensor] = None, check_status: bool = False) -> Tensor:
    """Attention of a batch's new tokens over the pages of their requests.

    q [T,H_q,128] (fp16 / bf16, the pages' dtype, after rotation); k_pages, v_pages [n_pages,H_kv,page_size,128] with
    page_size a power of two from 16 to 1024 and up to 16 query heads a KV head; block_tables int32 [S,width], q_start
    int32 [S+1], kv_lens int32 [S] (as :func:`build_block_tables` leaves them: q_start must not fall).  The last ``q_start[i+1]-q_start[i]`` of
    request i's ``kv_lens[i]`` tokens are the new ones, whose keys and values are in the pages already; where q_start goes past
    T, the rows that q has keep the places they have among these (a step with fewer token places than tokens).  A token
    sees its request's tokens up to itself; with ``window`` > 0 only the last ``window`` of them (itself included)
    and the request's first ``sinks``.  Tokens whose page is missing (an entry outside the pages) are not seen, and what
    stands in masked places does not matter, whatever it is.  A token that sees nothing gets zeros.

    max_new: the longest chunk of the batch (default T), which chooses the kernel: a hint, results do not depend on it but for their rounding.
    window and sinks from 2^30 on count as 2^30.
    scale: of the scores, positive, default 1/sqrt(128).  check_status: wait for the kernels and raise if one of their
    bounded waits ran out or q_start falls, in which case the results are invalid (where q_start falls nothing is computed: an
    ``out`` that the call allocates is zero, a given one as it was); without it the call returns at once.
    Returns ``out`` [T,H_q,128] in q's dtype.  Tokens in front of the first request's and behind the
    last one's are padding: zero in an ``out`` that the
    call allocates, left as they were in one that it is given (which must not share memory with q).  ``out_partial`` float32 [T*H_q,132] receives
    un-normalised records ``(m, l, -, -, o[128])`` instead, for :func:`rdkv_b200.decode.lse_combine` (rows of no request: as they were);
    their o is a sum in 32 bits of values times weights that were rounded to q's type, so it is as good as a result before its own rounding, not
    as 32 bits."""
    window, sinks = int(window), int(sinks)                # (numbers: a key must not go by the identity of a tensor that holds one)
    max_new, scale = None if max_new is None else int(max_new), None if scale is None else float(scale)
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.get_device(), v_pages.shape,
           v_pages.stride(), v_pages.dtype, v_pages.get_device(), block_tables.shape, block_tables.stride(), block_tables.dtype,
           block_tables.get_device(), q_start.shape, q_start.stride(), q_start.dtype, q_start.get_device(), kv_lens.shape, kv_lens.stride(),
           kv_lens.dtype, kv_lens.get_device(), max_new, window, sinks, scale)
    call = _ATTENTION_CALLS.get(key)
    if call is None:
        call = _ATTENTION_CALLS.remember(key, _attention_check(q, k_pages, v_pages, block_tables, q_start, kv_lens, max_new, window, sinks, scale))
    args, direct, n_ws, index, fields, dense = call
    if not direct or q.data_ptr() & 15:                    # (rows that no 16-byte or TMA copy can fetch)
        q, dense = q.clone(memory_format=torch.contiguous_format), True
        fields = PagedAttentionArgs.from_buffer_copy(fields)
        fields.q_tok_stride, fields.q_head_stride = q.stride()[:2]
        args = C.addressof(fields)
    k_ptr, v_ptr = k_pages.data_ptr(), v_pages.data_ptr()
    if (k_ptr | v_ptr) & 15:
        raise ValueError("k_pages and v_pages must start on 16 bytes")
    if out_partial is None:
        zero = 0
        if out is None:
            out, zero = empty_rows(q, dense), 1
        else:
            require_cuda(out, "out")
            if (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1 or out.data_ptr() % 16
                    or out.stride(0) % 8 or out.stride(1) % 8):
                raise ValueError(f"out must be {q.dtype} {tuple(q.shape)} on {q.device} with contiguous rows on 16 bytes")
            separate_rows(out, "out")
            if out.numel() > 0 and not apart(out, out.data_ptr(), footprint(out), q, q.data_ptr(), footprint(q)):
                raise ValueError("out must not share memory with q")
        os, out_ptr, rec_ptr = out.stride(), out.data_ptr(), None
    else:
        if out is not None:
            raise ValueError("either out or out_partial")
        require_cuda(out_partial, "out_partial")
        if (out_partial.dtype != torch.float32 or not out_partial.is_contiguous() or out_partial.device != q.device
                or out_partial.numel() != q.shape[0] * q.shape[1] * PARTIAL_STRIDE or out_partial.data_ptr() & 15):
            raise ValueError(f"out_partial must be contiguous float32 [{q.shape[0] * q.shape[1]},{PARTIAL_STRIDE}] on {q.device}, on 16 bytes")
        os, out_ptr, rec_ptr, zero = (0, 0), None, out_partial.data_ptr(), 0
    ws = kv_lens.new_empty(n_ws)
    status = lib().rdkv_paged_attention(args, q.data_ptr(), k_ptr, v_ptr, block_tables.data_ptr(), q_start.data_ptr(), kv_lens.data_ptr(),
                                        out_ptr, os[0], os[1], zero, rec_ptr, ws.data_ptr(), 4 * n_ws, raw_stream(index))
    if status:
        check(status, "rdkv_paged_attention")
    if check_status and n_ws > 0:
        trouble = int(ws[:lib().rdkv_paged_attention_status_words()].max())
        if trouble & 2:
            raise ValueError("q_start must not fall: nothing was computed")
        if trouble:
            raise RuntimeError("rdkv_paged_attention: a device-side wait ran out; the results are invalid")
    return out if out_partial is None else out_partial


def _attention_check(q, k_pages, v_pages, block_tables, q_start, kv_lens, max_new, window, sinks, scale):
    require_cuda(q, "q")
    _check_pages(k_pages, v_pages, False)
    n_pages, H_kv, page_size, _ = k_pages.shape
    if q.dim() != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be [T,H_q,{HEAD_DIM}], got {tuple(q.shape)}")
    T, H_q, _ = q.shape
    if q.dtype != k_pages.dtype or q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"q and the pages must both be fp16 or both bf16, got {q.dtype} and {k_pages.dtype}")
    if H_kv < 1 or H_q % H_kv or not 1 <= H_q // H_kv <= 16:
        raise ValueError(f"{H_q} query heads over {H_kv} KV heads: 1 to 16 each are supported")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
    _int32(block_tables, "block_tables", 2); _int32(q_start, "q_start", 1); _int32(kv_lens, "kv_lens", 1)
    S = kv_lens.shape[0]
    if block_tables.shape[0] != S or q_start.shape[0] != S + 1:
        raise ValueError(f"block_tables must have {S} rows and q_start {S + 1} elements")
    if S > MAX_REQUESTS:
        raise ValueError(f"{S} requests: at most {MAX_REQUESTS}")
    fits_32_bits(T=T, H_q=H_q, n_pages=n_pages, width=block_tables.shape[1])
    if window < 0 or sinks < 0 or (sinks > 0 and window == 0):
        raise ValueError("window and sinks must not be negative, and sinks need a window")
    scale = HEAD_DIM ** -0.5 if scale is None else scale
    if not 1e-30 < scale < 1e30:                           # (an ordinary number in 32 bits)
        raise ValueError(f"scale must be positive and finite, got {scale}")
    max_new = T if max_new is None else min(max_new, T)
    if max_new < 0:
        raise ValueError("max_new must not be negative")
    ks, vs = k_pages.stride()[:3], v_pages.stride()[:3]
    if any(x % 8 for x in ks + vs):
        raise ValueError("k_pages and v_pages must have strides of whole 16 bytes")
    _same_device(q.device, k_pages=k_pages, v_pages=v_pages, block_tables=block_tables, q_start=q_start, kv_lens=kv_lens)
    direct = q.stride(2) == 1 and all(st % 8 == 0 and (st > 0 or n == 1) for n, st in zip(q.shape[:2], q.stride()))
    n_ws = -(-lib().rdkv_paged_attention_workspace(S, T, H_q, H_kv, max_new) // 4)
    args = PagedAttentionArgs(
        q_tok_stride=q.stride(0), q_head_stride=q.stride(1), k_page_stride=ks[0], k_head_stride=ks[1], k_row_stride=ks[2], v_page_stride=vs[0],
        v_head_stride=vs[1], v_row_stride=vs[2], table_stride=block_tables.stride(0), dtype=q_dtype_tag(q), n_tokens=T, H_q=H_q, H_kv=H_kv,
        n_pages=n_pages, page_size=page_size, width=block_tables.shape[1], n_requests=S, max_new=max_new,
        window=min(window, 1 << 30), sinks=min(sinks, 1 << 30), scale=scale)
    return C.addressof(args), direct, n_ws, q.device.index, args, q.is_contiguous()
