"""Rotary position embedding of a decode step's query and key rows.

Drop-in for the reference's ``fused_rope`` (obkv_accel/triton_rope.py:111-138): same name,
arguments and in-place behaviour.  Inside a decode step the rotation is part of the attention
launch (:func:`rdkv_b200.decode.packed_decode_attention` with ``rope=``); this call is for
callers that keep the two steps apart.  :func:`rope_axes` rotates the rows of many tokens, each by
its own position on one to four axes.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch
from torch import Tensor

from ._lib import (HEAD_DIM, CallCache, RopeAxesArgs, apart, check, fits_32_bits, footprint, lib, ptr, q_dtype_tag, raw_stream, require_cuda,
                   separate_rows, stream_ptr)


def fused_rope(q: Tensor, k: Tensor, cos_half: Tensor, sin_half: Tensor):
    """Rotate q [H_q,128] and k [H_kv,128] (fp16 / bf16 / fp32) in place, half format:
    (x[i], x[i+64]) -> (x[i]·cos[i] − x[i+64]·sin[i], x[i+64]·cos[i] + x[i]·sin[i]) with fp32
    arithmetic; cos_half / sin_half [64].  Returns (q, k).  One launch."""
    for name, t in (("q", q), ("k", k), ("cos_half", cos_half), ("sin_half", sin_half)):
        require_cuda(t, name)
    if q.dim() != 2 or k.dim() != 2 or q.shape[1] != HEAD_DIM or k.shape[1] != HEAD_DIM:
        raise ValueError(f"q and k must be [heads,{HEAD_DIM}], got {tuple(q.shape)} and {tuple(k.shape)}")
    if cos_half.shape[0] != HEAD_DIM // 2 or sin_half.shape[0] != HEAD_DIM // 2 or cos_half.dtype != sin_half.dtype:
        raise ValueError(f"cos_half and sin_half must hold {HEAD_DIM // 2} values of one dtype")
    if q.stride(1) != 1 or k.stride(1) != 1:
        raise ValueError("q and k rows must be contiguous")
    cos_half, sin_half = cos_half.contiguous(), sin_half.contiguous()
    check(lib().rdkv_rope(ptr(q), q_dtype_tag(q), q.shape[0], q.stride(0), ptr(k), q_dtype_tag(k), k.shape[0],
                          k.stride(0), ptr(cos_half), ptr(sin_half), q_dtype_tag(cos_half), stream_ptr(q.device)),
          "rdkv_rope")
    return q, k


_AXES_TAG = {torch.int32: 0, torch.int64: 1}


def axes_check(positions: Tensor, inv_freq: Tensor, sections: Optional[Sequence[int]], T: int, dev):
    """The fields of a call's arguments that say how it rotates, by name."""
    half = HEAD_DIM // 2
    require_cuda(positions, "positions"); require_cuda(inv_freq, "inv_freq")
    n_axes = positions.shape[0] if positions.dim() == 2 else 1
    if positions.dim() not in (1, 2) or positions.shape[-1] != T or not 1 <= n_axes <= 4 or (T > 1 and positions.stride(-1) != 1):
        raise ValueError(f"positions must be [{T}] or [1 to 4 axes,{T}] with contiguous rows, got {tuple(positions.shape)}")
    if positions.dtype not in _AXES_TAG:
        raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    if inv_freq.dtype != torch.float32 or tuple(inv_freq.shape) != (half,) or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must be a contiguous float32 tensor of {half} elements")
    if positions.device != dev or inv_freq.device != dev:
        raise ValueError(f"positions and inv_freq must live on {dev}")
    if sections is None:
        if n_axes != 1:
            raise ValueError("positions of several axes need sections")
        sections = (half,)
    if any(int(n) != n or n < 0 for n in sections) or sum(sections) != half or len(sections) != n_axes:
        raise ValueError(f"sections must be {n_axes} whole numbers (one an axis) that add up to {half}, got {tuple(sections)}")
    return dict(axis_stride=0 if n_axes == 1 else positions.stride(0), positions_64=_AXES_TAG[positions.dtype], n_axes=n_axes,
                sections=(C.c_int32 * 4)(*(int(n) for n in sections)))


def empty_rows(t: Tensor, dense: bool) -> Tensor:
    """A contiguous tensor like ``t`` (``dense``: t is contiguous itself, and the shorter way leads there: 1.3 us for 2.4)."""
    return torch.empty_like(t) if dense else t.new_empty(t.shape)


def plain_sections(sections: Sequence[int]) -> tuple:
    """Sections as numbers (a key must not go by the identity of tensors that hold them)."""
    for n in sections:
        if type(n) is not int:
            return tuple(map(float, sections))
    return tuple(sections)


_ROPE_CALLS = CallCache()


def rope_axes(q: Tensor, k: Tensor, positions: Tensor, inv_freq: Tensor, *, sections: Optional[Sequence[int]] = None,
              q_out: Optional[Tensor] = None, k_out: Optional[Tensor] = None):
    """Rotate q [T,H_q,128] and k [T,H_kv,128] (both fp16, bf16 or fp32) by the tokens' positions, half format as
    :func:`fused_rope`.  One launch.

    positions [T], or [axes,T] with 1 to 4 axes (time, height, width of images and video), int32 / int64; inv_freq
    float32 [64]: the angle of frequency j is ``position * inv_freq[j]``, whose whole turns are taken off exactly, so that far positions
    lose nothing (up to 2^53).  sections: how many of the 64 frequencies each axis owns, in order (text
    with one axis: all of them).  Returns (q_out, k_out): new tensors, or the given ones, which may be q and k
    themselves (and must share no other memory with them)."""
    if sections is not None:
        sections = plain_sections(sections)
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), positions.shape, positions.stride(),
           positions.dtype, positions.get_device(), inv_freq.shape, inv_freq.stride(), inv_freq.dtype, inv_freq.get_device(),
           sections, None if q_out is None else (q_out.shape, q_out.stride(), q_out.dtype, q_out.get_device()),
           None if k_out is None else (k_out.shape, k_out.stride(), k_out.dtype, k_out.get_device()))
    call = _ROPE_CALLS.get(key)
    if call is None:
        call = _ROPE_CALLS.remember(key, _rope_check(q, k, positions, inv_freq, sections, q_out, k_out))
    args, _, index, dense, marks = call
    if marks is not None:
        _rope_apart(q, k, q_out, k_out, *marks)
    if q_out is None:
        q_out = empty_rows(q, dense)
    if k_out is None:
        k_out = empty_rows(k, dense)
    status = lib().rdkv_rope_axes(args, q.data_ptr(), q_out.data_ptr(), k.data_ptr(), k_out.data_ptr(), positions.data_ptr(),
                                  inv_freq.data_ptr(), raw_stream(index))
    if status:
        check(status, "rdkv_rope_axes")
    return q_out, k_out


def _rope_apart(q, k, q_out, k_out, q_mark, k_mark, qo_mark, ko_mark, q_like, k_like):
    """Refuses results that share memory with rows that are still to be read or with one another: each may be its own input, row for row
    (``_like``: strides are the same), and nothing else."""
    pq, pk = q.data_ptr(), k.data_ptr()
    pqo, pko = None if q_out is None else q_out.data_ptr(), None if k_out is None else k_out.data_ptr()
    q_in, k_in = q_like and pqo == pq, k_like and pko == pk
    if not ((q_out is None or ((q_in or apart(q_out, pqo, qo_mark, q, pq, q_mark)) and (k_in or apart(q_out, pqo, qo_mark, k, pk, k_mark))))
            and (k_out is None or ((k_in or apart(k_out, pko, ko_mark, k, pk, k_mark)) and (q_in or apart(k_out, pko, ko_mark, q, pq, q_mark))))
            and (q_out is None or k_out is None or apart(q_out, pqo, qo_mark, k_out, pko, ko_mark))):
        raise ValueError("q_out and k_out may be q and k themselves, but must share no other memory with them or with one another")


def _rope_check(q, k, positions, inv_freq, sections, q_out, k_out):
    for name, t in (("q", q), ("k", k)):
        require_cuda(t, name)
        if t.dim() != 3 or t.shape[2] != HEAD_DIM or t.stride(2) != 1:
            raise ValueError(f"{name} must be [T,heads,{HEAD_DIM}] with contiguous rows, got {tuple(t.shape)}")
    T, dev = q.shape[0], q.device
    fits_32_bits(T=T, H_q=q.shape[1], H_kv=k.shape[1])
    if k.shape[0] != T or k.dtype != q.dtype or k.device != dev:
        raise ValueError("q and k must have the same tokens, dtype and device")
    for name, t, x in (("q_out", q_out, q), ("k_out", k_out, k)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != dev or t.stride(2) != 1):
            raise ValueError(f"{name} must have the shape, dtype and device of its input and contiguous rows")
        if t is not None:
            separate_rows(t, name)
    (q0, q1), (k0, k1) = q.stride()[:2], k.stride()[:2]
    qo = (q.shape[1] * HEAD_DIM, HEAD_DIM) if q_out is None else q_out.stride()
    ko = (k.shape[1] * HEAD_DIM, HEAD_DIM) if k_out is None else k_out.stride()
    args = RopeAxesArgs(q_tok_stride=q0, q_head_stride=q1, q_out_tok_stride=qo[0], q_out_head_stride=qo[1], k_tok_stride=k0, k_head_stride=k1,
                        k_out_tok_stride=ko[0], k_out_head_stride=ko[1], H_q=q.shape[1], H_kv=k.shape[1], dtype=q_dtype_tag(q), n_tokens=T,
                        **axes_check(positions, inv_freq, sections, T, dev))
    marks = None
    if q_out is not None or k_out is not None:
        marks = (footprint(q), footprint(k), q_out is not None and footprint(q_out), k_out is not None and footprint(k_out),
                 q_out is not None and q_out.stride() == q.stride(), k_out is not None and k_out.stride() == k.stride())
    return C.addressof(args), args, dev.index, q.is_contiguous() and k.is_contiguous(), marks
