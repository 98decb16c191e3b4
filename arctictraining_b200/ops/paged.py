# SPDX-License-Identifier: Apache-2.0
"""Operators of the paged generation cache.

A cache is ``pages [P, heads, page, dim]``: page ``p`` holds ``page`` consecutive positions of one sequence.  Its elements
have the model's type, or are e4m3 with one fp32 scale of 0 or more per position and head (``[P, heads, page]``).  ``page_table [B, W]``
(int32) names the pages of every sequence in order; an id outside ``[0, P)`` stands for no page: writes to it are dropped and
reads skip it.  The heads, positions and elements of a page are dense; pages may lie further apart (slices of a larger tensor),
keys and values equally far.  ``starts [B]`` (int32) are the tokens that a sequence had before the call; its new token ``j`` stands at
position ``starts + j``.  ``counts [B]`` (int32) limits the new tokens of a padded batch: token ``j`` of a sequence takes part
when ``j < counts`` (default: all).  Places of one call must differ: two tokens written to one place leave either of them.

bf16 / fp16 tensors on a GPU use the kernels of ``csrc/paged_cache.cu`` and ``csrc/paged_attention.cu`` (widths that are
multiples of 16: heads up to 256, latents up to 512 with a rotary part up to 64); other types, widths and the CPU use
:mod:`.reference`.  Nothing here is differentiable: inputs that need a gradient are refused.  Calls on the kernels do not wait
for the GPU and can be captured into a CUDA graph after a first call outside of it; the page table, starts and counts are read
when the graph runs.  Rows, tables and lengths of layouts other than these, and on the kernels pages that do not start on 16 bytes,
are refused; queries, keys and values that are not aligned to 16 bytes are copied.  Latent attention of many heads waits inside its
kernel for a bounded time only: a wait that ran out leaves a code in the device's error word (:mod:`..comm.errors`), which the
training engine and ``models.generation.generate`` read.
"""

from __future__ import annotations

import os
from typing import Optional
from typing import Tuple

import torch

from . import _ext
from . import reference as ref
from .functional import _count

_HALF = (torch.bfloat16, torch.float16)
_LARGEST = torch.finfo(torch.float32).max


def _use_kernels(t: torch.Tensor) -> bool:
    """As in :mod:`.functional`, without its questions to the driver once the library is loaded: a decoding step makes this
    call in every layer."""
    return t.is_cuda and ((_ext._loaded is True and "ATB200_DISABLE_KERNELS" not in os.environ) or _ext.available())


def _refuse(cond: bool, what: str) -> None:
    if cond:
        raise ValueError(what)


def _check_scale(op: str, scale: float) -> None:
    _refuse(not abs(scale) <= _LARGEST, f"{op}: scale must be a finite 32-bit number")


def _no_grad(op: str, *tensors: torch.Tensor) -> None:
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if t.requires_grad:
            raise ValueError(f"{op}: the generation cache is not differentiable; call it under torch.no_grad()")


def _dense_inside(t: torch.Tensor) -> bool:
    """Whether every slice along the first dimension is dense (a dimension of one element may have any stride)."""
    step = 1
    for size, stride in zip(t.shape[:0:-1], t.stride()[:0:-1]):
        if size != 1 and stride != step:
            return False
        step *= size
    return True


def _check_pages(op: str, pages: torch.Tensor, scale: Optional[torch.Tensor], x: torch.Tensor) -> None:
    _refuse(pages.dim() != 4, f"{op}: pages must be [pages, heads, page, dim]")
    _refuse(pages.shape[2] < 1, f"{op}: a page holds at least one position")
    _refuse(pages.device != x.device, f"{op}: all tensors must be on one device")
    _refuse(not _dense_inside(pages), f"{op}: the heads, positions and elements of a page must be dense")
    if pages.dtype == torch.float8_e4m3fn:
        _refuse(scale is None, f"{op}: an e4m3 cache needs its scales")
        _refuse(scale.dtype != torch.float32 or scale.shape != pages.shape[:3], f"{op}: scales must be fp32 [pages, heads, page]")
        _refuse(not _dense_inside(scale), f"{op}: the scales of a page must be dense")
        _refuse(scale.device != x.device, f"{op}: all tensors must be on one device")
    else:
        _refuse(scale is not None, f"{op}: scales belong to an e4m3 cache")


def _check_table(op: str, table: torch.Tensor, lens: torch.Tensor, counts: Optional[torch.Tensor], pages: torch.Tensor, B: int) -> None:
    _refuse(table.dim() != 2 or table.shape[0] != B or table.dtype != torch.int32, f"{op}: page_table must be int32 [batch, pages]")
    _refuse(table.shape[1] > 1 and table.stride(1) != 1, f"{op}: the rows of page_table must be dense")
    for t, name in ((lens, "starts / lengths"), (counts, "counts")):
        if t is not None:
            _refuse(t.shape != (B,) or t.dtype != torch.int32 or not t.is_contiguous(), f"{op}: {name} must be dense int32 [batch]")
            _refuse(t.device != pages.device, f"{op}: all tensors must be on one device")
    _refuse(table.device != pages.device, f"{op}: all tensors must be on one device")
    _refuse(table.shape[1] * pages.shape[2] >= 2**31 - 2**20, f"{op}: a sequence holds fewer than 2^31 positions")


def _check_cos_sin(op: str, cos: torch.Tensor, sin: torch.Tensor, shape: Tuple[int, int, int], x: torch.Tensor) -> None:
    _refuse(cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.shape != shape or sin.shape != shape,
            f"{op}: cos and sin must be fp32 [batch, new tokens, rotary width / 2]")
    _refuse(cos.device != x.device or sin.device != x.device, f"{op}: all tensors must be on one device")


def paged_kv_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: Optional[torch.Tensor] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Rotates the new tokens' queries ``q [B, S, Hq, D]`` and keys ``k [B, S, Hkv, D]`` (rotate-half, ``cos / sin
    [B, S, D/2]`` fp32), writes keys and values to their places in the cache and returns the rotated queries.  q, k and v may
    be strided views of a fused projection."""
    op = "paged_kv_append"
    _no_grad(op, q, k, v)
    if _use_kernels(q) and q.dtype in _HALF and q.dim() == 4 and q.shape[-1] % 16 == 0 and 0 < q.shape[-1] <= 256:
        _count()
        return _ext.ops().paged_kv_append(q, k, v, cos, sin, k_pages, v_pages, page_table, starts, counts, k_scale, v_scale)
    _refuse(q.dim() != 4 or k.dim() != 4 or v.dim() != 4, f"{op}: q, k and v must be [batch, new tokens, heads, dim]")
    B, S, _, D = q.shape
    _refuse(k.shape[:2] != (B, S) or k.shape[3] != D or v.shape != k.shape, f"{op}: q, k and v differ in shape")
    _refuse(D % 2 != 0, f"{op}: dim must be even")
    _refuse(k.dtype != q.dtype or v.dtype != q.dtype or not q.is_floating_point(), f"{op}: q, k and v must be of one floating type")
    _refuse(k.device != q.device or v.device != q.device, f"{op}: all tensors must be on one device")
    _check_cos_sin(op, cos, sin, (B, S, D // 2), q)
    _check_pages(op, k_pages, k_scale, q)
    _check_pages(op, v_pages, v_scale, q)
    _refuse(k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype, f"{op}: k_pages and v_pages differ")
    _refuse(k_pages.shape[1] != k.shape[2] or k_pages.shape[3] != D, f"{op}: the cache has other heads or another dim than k")
    _refuse(k_scale is None and k_pages.dtype != q.dtype, f"{op}: the cache must have the inputs' type or be e4m3")
    _check_table(op, page_table, starts, counts, k_pages, B)
    return ref.paged_kv_append(q, k, v, cos, sin, k_pages, v_pages, page_table, starts, counts, k_scale, v_scale)


def _latent_widths_ok(latent: int, rope: int) -> bool:
    return latent % 16 == 0 and 0 < latent <= 512 and rope % 16 == 0 and 0 < rope <= 64


def paged_latent_append(
    q_pe: torch.Tensor,
    kv_a: torch.Tensor,
    norm_weight: torch.Tensor,
    eps: float,
    cos: torch.Tensor,
    sin: torch.Tensor,
    pages: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: Optional[torch.Tensor] = None,
    page_scale: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Multi-head latent attention's cache write: of ``kv_a [B, S, R + rope]`` the latent is RMS-normalised with
    ``norm_weight [R]``, the shared key rotated, and both written as one row of ``pages [P, 1, page, R + rope]``.  Returns
    the queries' rotary part ``q_pe [B, S, H, rope]``, rotated."""
    op = "paged_latent_append"
    _no_grad(op, q_pe, kv_a, norm_weight)
    if _use_kernels(q_pe) and q_pe.dtype in _HALF and q_pe.dim() == 4 and _latent_widths_ok(norm_weight.numel(), q_pe.shape[-1]):
        _count()
        return _ext.ops().paged_latent_append(q_pe, kv_a, norm_weight, eps, cos, sin, pages, page_table, starts, counts, page_scale)
    _refuse(q_pe.dim() != 4 or kv_a.dim() != 3,
            f"{op}: q_pe must be [batch, new tokens, heads, rotary] and kv_a [batch, new tokens, latent + rotary]")
    B, S, _, rope = q_pe.shape
    _refuse(norm_weight.dim() != 1 or kv_a.shape != (B, S, norm_weight.numel() + rope), f"{op}: q_pe, kv_a and norm_weight differ in shape")
    _refuse(rope % 2 != 0, f"{op}: the rotary part must be even")
    _refuse(kv_a.dtype != q_pe.dtype or norm_weight.dtype != q_pe.dtype or not q_pe.is_floating_point(),
            f"{op}: q_pe, kv_a and norm_weight must be of one floating type")
    _refuse(kv_a.device != q_pe.device or norm_weight.device != q_pe.device, f"{op}: all tensors must be on one device")
    _check_cos_sin(op, cos, sin, (B, S, rope // 2), q_pe)
    _check_pages(op, pages, page_scale, q_pe)
    _refuse(pages.shape[1] != 1 or pages.shape[3] != kv_a.shape[2], f"{op}: a latent cache is [pages, 1, page, latent + rotary]")
    _refuse(page_scale is None and pages.dtype != q_pe.dtype, f"{op}: the cache must have the inputs' type or be e4m3")
    _check_table(op, page_table, starts, counts, pages, B)
    return ref.paged_latent_append(q_pe, kv_a, norm_weight, eps, cos, sin, pages, page_table, starts, counts, page_scale)


def paged_kv_read(
    k_pages: torch.Tensor,
    v_pages: Optional[torch.Tensor],
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    max_length: int,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    dtype: Optional[torch.dtype] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The first ``max_length`` positions of every sequence as dense ``[B, max_length, heads, dim]`` tensors of ``dtype``
    (the cache's own by default; bf16 for an e4m3 one), zeros from ``lengths`` on.  ``v_pages=None`` (a latent cache) reads one
    tensor."""
    op = "paged_kv_read"
    if dtype is None:
        dtype = torch.bfloat16 if k_pages.dtype == torch.float8_e4m3fn else k_pages.dtype
    if _use_kernels(k_pages) and dtype in _HALF and k_pages.dim() == 4 and k_pages.shape[-1] % 16 == 0 and 0 < k_pages.shape[-1] <= 2048:
        _count()
        k, v = _ext.ops().paged_read(k_pages, v_pages, page_table, lengths, max_length, k_scale, v_scale, dtype)
        return k, None if v_pages is None else v
    _refuse(max_length < 0, f"{op}: max_length must be 0 or more")
    out = []
    for pages, scale in ((k_pages, k_scale), (v_pages, v_scale)):
        if pages is None:
            out.append(None)
            continue
        _check_pages(op, pages, scale, k_pages)
        _refuse(pages.shape != k_pages.shape or pages.dtype != k_pages.dtype, f"{op}: k_pages and v_pages differ")
        _refuse(scale is None and pages.dtype != dtype, f"{op}: the cache must have the result's type or be e4m3")
        _refuse(page_table.dim() != 2, f"{op}: page_table must be int32 [batch, pages]")
        _check_table(op, page_table, lengths, None, pages, page_table.shape[0])
        out.append(ref.paged_read(pages, page_table, lengths, max_length, scale, dtype))
    return out[0], out[1]


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: Optional[torch.Tensor] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    window: Optional[int] = None,
) -> torch.Tensor:
    """Attention of the new tokens' (rotated) queries ``q [B, S, Hq, D]`` over the cache, their own keys included.  Query ``j``
    of a sequence sees the positions up to ``starts + j``, with ``window`` only the last ``window`` of them.  ``Hq`` is a
    multiple of the cache's heads.  A query that sees nothing (no page, ``j >= counts``) gets zeros."""
    op = "paged_attention"
    _no_grad(op, q)
    if window is not None:
        _refuse(window < 1, f"{op}: window must be positive")
        window = min(window, 2**31 - 1)  # longer than any sequence
    if scale is None:
        scale = q.shape[-1] ** -0.5
    _check_scale(op, scale)
    if _use_kernels(q) and q.dtype in _HALF and q.dim() == 4 and q.shape[-1] % 16 == 0 and 0 < q.shape[-1] <= 256:
        _count()
        return _ext.ops().paged_attention(q, k_pages, v_pages, page_table, starts, counts, k_scale, v_scale, scale, window or 0)
    _refuse(q.dim() != 4, f"{op}: q must be [batch, new tokens, heads, dim]")
    _check_pages(op, k_pages, k_scale, q)
    _check_pages(op, v_pages, v_scale, q)
    _refuse(k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype, f"{op}: k_pages and v_pages differ")
    _refuse(k_pages.stride(0) != v_pages.stride(0) or (k_scale is not None and k_scale.stride(0) != v_scale.stride(0)),
            f"{op}: the pages of keys and values must lie equally far apart")
    _refuse(k_pages.shape[1] == 0 or q.shape[2] % k_pages.shape[1] != 0, f"{op}: the query heads must be a multiple of the cache's heads")
    _refuse(k_pages.shape[3] != q.shape[3], f"{op}: the cache has another dim than q")
    _refuse(k_scale is None and k_pages.dtype != q.dtype, f"{op}: the cache must have the query's type or be e4m3")
    _check_table(op, page_table, starts, counts, k_pages, q.shape[0])
    return ref.paged_attention(q, k_pages, v_pages, page_table, starts, counts, k_scale, v_scale, scale, window)


def paged_latent_attention(
    q_latent: torch.Tensor,
    q_pe: torch.Tensor,
    pages: torch.Tensor,
    page_table: torch.Tensor,
    starts: torch.Tensor,
    counts: Optional[torch.Tensor] = None,
    page_scale: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Absorbed form of multi-head latent attention: all heads attend to the cache's rows ``[latent | rotary key]`` with
    queries ``[q_latent | q_pe]`` (``q_latent [B, S, H, R]``: the query's position-free part times the key half of the
    up-projection), and the result ``[B, S, H, R]`` is the weighted sum of latents, which the value half of the up-projection
    turns into heads.  ``scale`` is that of the expanded heads and has to be given."""
    op = "paged_latent_attention"
    _no_grad(op, q_latent, q_pe)
    _refuse(scale is None, f"{op}: scale must be given")
    _check_scale(op, scale)
    if _use_kernels(q_latent) and q_latent.dtype in _HALF and q_latent.dim() == 4 and _latent_widths_ok(q_latent.shape[-1], q_pe.shape[-1]):
        _count()
        return _ext.ops().paged_latent_attention(q_latent, q_pe, pages, page_table, starts, counts, page_scale, scale)
    _refuse(q_latent.dim() != 4 or q_pe.dim() != 4, f"{op}: q_latent and q_pe must be [batch, new tokens, heads, width]")
    _refuse(q_pe.shape[:3] != q_latent.shape[:3], f"{op}: q_latent and q_pe differ in shape")
    _refuse(q_pe.dtype != q_latent.dtype or not q_pe.is_floating_point(), f"{op}: q_latent and q_pe must be of one floating type")
    _refuse(q_pe.device != q_latent.device, f"{op}: all tensors must be on one device")
    _check_pages(op, pages, page_scale, q_latent)
    _refuse(pages.shape[1] != 1 or pages.shape[3] != q_latent.shape[3] + q_pe.shape[3], f"{op}: a latent cache is [pages, 1, page, latent + rotary]")
    _refuse(page_scale is None and pages.dtype != q_latent.dtype, f"{op}: the cache must have the query's type or be e4m3")
    _check_table(op, page_table, starts, counts, pages, q_latent.shape[0])
    return ref.paged_latent_attention(q_latent, q_pe, pages, page_table, starts, counts, page_scale, scale)
