# SPDX-License-Identifier: Apache-2.0
"""Plain PyTorch implementations of every fused op.

These are the oracle the CUDA kernels are tested against and the code path used on CPU (Gloo runs,
unit tests).  They compute in fp32 internally and return the input dtype.
"""

from __future__ import annotations

import math
from typing import Optional
from typing import Tuple

import torch
import torch.nn.functional as F

IGNORE_INDEX = -100


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    inv = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * inv * weight.float()).to(x.dtype)


def rope_cos_sin(
    position_ids: torch.Tensor, head_dim: int, theta: float, scaling: Optional[dict] = None
) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos/sin tables ``[..., head_dim/2]`` in fp32 for the given positions (rotate-half convention)."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=position_ids.device) / head_dim))
    if scaling and scaling.get("rope_type", scaling.get("type")) == "llama3":
        factor = scaling["factor"]
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        old_len = scaling["original_max_position_embeddings"]
        wavelen = 2 * math.pi / inv_freq
        smooth = ((old_len / wavelen) - low) / (high - low)
        scaled = torch.where(wavelen > old_len / low, inv_freq / factor, inv_freq)
        mid = (1 - smooth) * inv_freq / factor + smooth * inv_freq
        is_mid = (wavelen <= old_len / low) & (wavelen >= old_len / high)
        inv_freq = torch.where(is_mid, mid, scaled)
    amplitude = 1.0
    if scaling and scaling.get("rope_type", scaling.get("type")) == "yarn":
        inv_freq, amplitude = _yarn_inv_freq(inv_freq, head_dim, theta, scaling)
    ang = position_ids.float().unsqueeze(-1) * inv_freq
    if amplitude != 1.0:
        return ang.cos() * amplitude, ang.sin() * amplitude
    return ang.cos(), ang.sin()


def yarn_mscale(factor: float, mscale: float = 1.0) -> float:
    return 1.0 if factor <= 1 else 0.1 * mscale * math.log(factor) + 1.0


def _yarn_inv_freq(inv_freq: torch.Tensor, dim: int, theta: float, scaling: dict):
    """YaRN: frequencies whose wavelength fits ``beta_fast`` times into the original context keep their value, those
    fitting fewer than ``beta_slow`` times are divided by ``factor``, a linear ramp in between; cos/sin are scaled by
    ``mscale(factor, mscale) / mscale(factor, mscale_all_dim)``."""
    factor = float(scaling["factor"])
    orig = float(scaling.get("original_max_position_embeddings") or 4096)
    fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)

    def correction_dim(rotations: float) -> float:
        return dim * math.log(orig / (rotations * 2 * math.pi)) / (2 * math.log(theta))

    low = max(math.floor(correction_dim(fast)), 0)
    high = min(math.ceil(correction_dim(slow)), dim - 1)
    if low == high:
        high += 0.001
    ramp = ((torch.arange(dim // 2, dtype=torch.float32, device=inv_freq.device) - low) / (high - low)).clamp(0, 1)
    keep = 1.0 - ramp
    blended = inv_freq / factor * (1 - keep) + inv_freq * keep
    m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
    amplitude = yarn_mscale(factor, m) / yarn_mscale(factor, m_all) if (m and m_all) else yarn_mscale(factor)
    if scaling.get("attention_factor") is not None:
        amplitude = float(scaling["attention_factor"])
    return blended, float(amplitude)


def rope_apply(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, inverse: bool = False) -> torch.Tensor:
    """Rotate ``x [B, S, H, D]`` with ``cos/sin [B, S, D/2]``: pairs are ``(x[i], x[i + D/2])``."""
    d2 = x.shape[-1] // 2
    xf = x.float()
    x1, x2 = xf[..., :d2], xf[..., d2:]
    c = cos.unsqueeze(-2)
    s = sin.unsqueeze(-2)
    if inverse:
        s = -s
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1).to(x.dtype)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return (F.silu(gate.float()) * up.float()).to(gate.dtype)


GATE_UP_BLOCK = 64


def split_gate_up(gu: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Split a block-interleaved ``[..., 2I]`` tensor (64 gate columns, 64 up columns, ...) into halves."""
    shp = gu.shape
    v = gu.reshape(*shp[:-1], shp[-1] // (2 * GATE_UP_BLOCK), 2, GATE_UP_BLOCK)
    return v[..., 0, :].reshape(*shp[:-1], -1), v[..., 1, :].reshape(*shp[:-1], -1)


def swiglu_interleaved(gu: torch.Tensor) -> torch.Tensor:
    g, u = split_gate_up(gu)
    return swiglu(g, u)


def interleave_gate_up_rows(gate_w: torch.Tensor, up_w: torch.Tensor) -> torch.Tensor:
    """Build the fused ``[2I, H]`` weight whose output columns are block-interleaved (block = 64)."""
    inter, hidden = gate_w.shape
    assert inter % GATE_UP_BLOCK == 0, "intermediate size must be a multiple of 64"
    g = gate_w.reshape(inter // GATE_UP_BLOCK, 1, GATE_UP_BLOCK, hidden)
    u = up_w.reshape(inter // GATE_UP_BLOCK, 1, GATE_UP_BLOCK, hidden)
    return torch.cat((g, u), dim=1).reshape(2 * inter, hidden)


def deinterleave_gate_up_rows(fused: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    two_i, hidden = fused.shape
    v = fused.reshape(two_i // (2 * GATE_UP_BLOCK), 2, GATE_UP_BLOCK, hidden)
    return v[:, 0].reshape(-1, hidden).contiguous(), v[:, 1].reshape(-1, hidden).contiguous()


def segment_ids_from_cu(cu_seqlens: torch.Tensor, total: int) -> torch.Tensor:
    pos = torch.arange(total, device=cu_seqlens.device)
    return torch.bucketize(pos, cu_seqlens[1:], right=True)


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    causal: bool = True,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Causal GQA attention.  ``q [B,S,Hq,D]``, ``k/v [B,S,Hkv,D]``.  With ``cu_seqlens`` (``B == 1``)
    tokens attend only inside their own packed sample."""
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    qf = q.float().transpose(1, 2)
    kf = k.float().transpose(1, 2).repeat_interleave(Hq // Hkv, dim=1)
    vf = v.float().transpose(1, 2).repeat_interleave(Hq // Hkv, dim=1)
    scores = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    mask = torch.ones(S, S, dtype=torch.bool, device=q.device)
    if causal:
        mask = torch.tril(mask)
    if cu_seqlens is not None:
        seg = segment_ids_from_cu(cu_seqlens, S)
        mask = mask & (seg[:, None] == seg[None, :])
    scores = scores.masked_fill(~mask, float("-inf"))
    out = torch.matmul(torch.softmax(scores, dim=-1), vf)
    return out.transpose(1, 2).to(q.dtype)


def cross_entropy_sum(logits: torch.Tensor, labels: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sum of token losses (fp32) and the number of labels that are not ``-100``."""
    lf = logits.float()
    loss = F.cross_entropy(lf, labels, ignore_index=IGNORE_INDEX, reduction="sum")
    return loss, (labels != IGNORE_INDEX).sum()


def adamw_step(
    master: torch.Tensor,
    grad: torch.Tensor,
    exp_avg: torch.Tensor,
    exp_avg_sq: torch.Tensor,
    lr: float,
    beta1: float,
    beta2: float,
    eps: float,
    weight_decay: float,
    step: int,
    grad_scale: float = 1.0,
    out_lp: Optional[torch.Tensor] = None,
) -> None:
    """Decoupled-weight-decay Adam on flat tensors, in place; optionally writes a low-precision copy."""
    g = grad.float() * grad_scale
    m = exp_avg.float().mul_(beta1).add_(g, alpha=1 - beta1)
    v = exp_avg_sq.float().mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1**step
    bc2 = 1 - beta2**step
    p = master.float()
    p.mul_(1 - lr * weight_decay)
    denom = (v / bc2).sqrt_().add_(eps)
    p.addcdiv_(m / bc1, denom, value=-lr)
    master.copy_(p)
    exp_avg.copy_(m)
    exp_avg_sq.copy_(v)
    if out_lp is not None:
        out_lp.copy_(p)


def topk_gating(logits: torch.Tensor, top_k: int, normalize: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Softmax over all experts (fp32), top-k (ties → lower index), optional renormalisation.

    Returns ``probs [T,E]`` fp32, ``scores [T,K]`` fp32, ``experts [T,K]`` int64.
    """
    probs = torch.softmax(logits.float(), dim=-1)
    # stable descending sort gives the lower expert index on ties
    order = torch.sort(probs, dim=-1, descending=True, stable=True).indices[:, :top_k]
    scores = torch.gather(probs, 1, order)
    if normalize:
        scores = scores / scores.sum(-1, keepdim=True)
    return probs, scores, order


# ------------------------------------------------------------------------------------------------ paged generation cache
E4M3_MAX = 448.0
E4M3_TINY = 2.0**-100


def quantize_rows_e4m3(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of ``x [..., D]`` as e4m3 values and one fp32 scale each: largest magnitude / 448 (at least 2^-100 / 448, so
    that a row of zeros has one too)."""
    xf = x.float()
    scale = xf.abs().amax(-1).clamp(min=E4M3_TINY) / E4M3_MAX
    return (xf * (1.0 / scale).unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _paged_slots(page_table, starts, counts, S: int, pages: torch.Tensor):
    """(written, page id, offset), each ``[B, S]``, of the new tokens' places."""
    P, page = pages.shape[0], pages.shape[2]
    B, W = page_table.shape
    j = torch.arange(S, device=pages.device).view(1, S)
    pos = starts.long().view(B, 1) + j
    ok = (starts.view(B, 1) >= 0) & (pos < W * page)
    if counts is not None:
        ok = ok & (j < counts.view(B, 1))
    if W == 0:
        return ok, pos, pos
    pid = torch.gather(page_table.long(), 1, (pos // page).clamp(0, W - 1))
    return ok & (pid >= 0) & (pid < P), pid, pos % page


def _paged_write(pages, scales, rows, page_table, starts, counts) -> None:
    ok, pid, off = _paged_slots(page_table, starts, counts, rows.shape[1], pages)
    pid, off, rows = pid[ok], off[ok], rows[ok]
    if scales is None:
        pages[pid, :, off] = rows.to(pages.dtype)
    else:
        values, sc = quantize_rows_e4m3(rows)
        pages.view(torch.uint8)[pid, :, off] = values.view(torch.uint8)
        scales[pid, :, off] = sc


def _paged_gather(pages, scales, page_table) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached rows in fp32 ``[B, H, W * page, D]`` and which of them lie on a page that exists ``[B, W * page]``."""
    P, H, page, D = pages.shape
    B, W = page_table.shape
    if P == 0 or W == 0:
        return (torch.zeros(B, H, W * page, D, device=pages.device),
                torch.zeros(B, W * page, device=pages.device, dtype=torch.bool))
    ids = page_table.long()
    held = (ids >= 0) & (ids < P)
    ids = ids.clamp(0, P - 1)
    if scales is None:
        x = pages[ids].float()
    else:
        x = pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float() * scales[ids].unsqueeze(-1)
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, W * page, D), held.repeat_interleave(page, dim=1)


def paged_kv_append(q, k, v, cos, sin, k_pages, v_pages, page_table, starts, counts=None, k_scale=None, v_scale=None):
    d2 = q.shape[-1] // 2
    c, s = cos.unsqueeze(2), sin.unsqueeze(2)

    def turn(x):
        x1, x2 = x[..., :d2].float(), x[..., d2:].float()
        return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)

    _paged_write(k_pages, k_scale, turn(k), page_table, starts, counts)
    _paged_write(v_pages, v_scale, v.float(), page_table, starts, counts)
    return turn(q).to(q.dtype)


def paged_latent_append(q_pe, kv_a, norm_weight, eps, cos, sin, pages, page_table, starts, counts=None, page_scale=None):
    R = norm_weight.shape[0]
    latent = kv_a[..., :R].float()
    latent = latent * torch.rsqrt(latent.pow(2).mean(-1, keepdim=True) + eps) * norm_weight.float()
    k_pe = rope_apply(kv_a[..., R:].float().unsqueeze(2), cos, sin)
    _paged_write(pages, page_scale, torch.cat((latent.unsqueeze(2), k_pe), dim=-1), page_table, starts, counts)
    return rope_apply(q_pe, cos, sin)


def paged_read(pages, page_table, lengths, max_length: int, page_scale, dtype) -> torch.Tensor:
    x, held = _paged_gather(pages, page_scale, page_table)
    B, H, L, D = x.shape
    n = min(max_length, L)
    held = held[:, :n] & (torch.arange(n, device=pages.device).view(1, n) < lengths.view(B, 1))
    out = torch.zeros(B, max_length, H, D, device=pages.device, dtype=dtype)
    out[:, :n] = torch.where(held.view(B, n, 1, 1), x[:, :, :n].transpose(1, 2), torch.zeros((), device=pages.device)).to(dtype)
    return out


def _paged_softmax_product(q, k, v, held, starts, counts, scale: float, window) -> torch.Tensor:
    """``q [B, S, Hq, D]`` against fp32 ``k / v [B, Hkv, L, .]``; a query that sees nothing gets zeros."""
    B, S, Hq, _ = q.shape
    Hkv, L = k.shape[1:3]
    if L == 0 or q.numel() == 0:
        return torch.zeros(B, S, Hq, v.shape[-1], device=q.device, dtype=q.dtype)
    at = torch.arange(L, device=q.device).view(1, 1, L)
    j = torch.arange(S, device=q.device).view(1, S, 1)
    mine = starts.long().view(B, 1, 1) + j
    seen = (at <= mine) & held.view(B, 1, L)
    if window:
        seen = seen & (at > mine - window)
    if counts is not None:
        seen = seen & (j < counts.view(B, 1, 1))
    any_query = seen.any(1).view(B, 1, L, 1)  # values that no query sees may be anything, NaN too
    v = torch.where(any_query, v, torch.zeros((), device=v.device, dtype=v.dtype))
    qf = q.float().view(B, S, Hkv, Hq // Hkv, -1).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(qf, k.unsqueeze(2).transpose(-1, -2)) * scale
    scores = scores.masked_fill(~seen.view(B, 1, 1, S, L), float("-inf"))
    p = torch.softmax(scores, dim=-1).masked_fill(~seen.any(-1).view(B, 1, 1, S, 1), 0.0)
    finite = torch.isfinite(v)
    o = torch.matmul(p, torch.where(finite, v, 0.0).unsqueeze(2))
    # infinities and NaN reach the queries that see them, and no others (0 times them is no 0)
    for t in torch.nonzero(~finite.all(-1).all(1).all(0)).flatten().tolist():
        rest = torch.where(finite[:, :, t], 0.0, v[:, :, t]).view(B, Hkv, 1, 1, -1)
        o = o + torch.where(seen[:, :, t].view(B, 1, 1, S, 1), p[..., t : t + 1] * rest, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, S, Hq, -1).to(q.dtype)


def paged_attention(q, k_pages, v_pages, page_table, starts, counts, k_scale, v_scale, scale: float, window) -> torch.Tensor:
    k, held = _paged_gather(k_pages, k_scale, page_table)
    v, _ = _paged_gather(v_pages, v_scale, page_table)
    return _paged_softmax_product(q, k, v, held, starts, counts, scale, window)


def paged_latent_attention(q_latent, q_pe, pages, page_table, starts, counts, page_scale, scale: float) -> torch.Tensor:
    k, held = _paged_gather(pages, page_scale, page_table)
    return _paged_softmax_product(torch.cat((q_latent, q_pe), dim=-1), k, k[..., : q_latent.shape[-1]], held, starts, counts,
                                  scale, None)
