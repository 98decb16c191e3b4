# SPDX-License-Identifier: Apache-2.0
"""Paged key/value cache for generation.

Keys and values live in pages of ``page`` positions that are handed to sequences as they grow, so a new token costs one row
written instead of a copy of the whole cache.  Rows keep the model's type, or are stored as e4m3 with one scale per position
and head (half the memory and half the traffic of a decoding step).  Multi-head latent attention stores its 576-wide latent
row instead of expanded heads.  The tensors are read and written by the ``ops.paged_*`` operators.
"""

from __future__ import annotations

from typing import List
from typing import Optional
from typing import Tuple

import torch
import torch.nn.functional as F

from .. import ops
from .arch import ArchConfig


class PagedKVCache:
    """``heads`` rows of ``dim`` elements per layer and position, for keys and for values; ``latent=True``: one joint row
    ``[latent | rotary key]`` instead.  ``num_pages`` pages are shared by ``batch`` sequences of up to ``max_length`` positions
    (default: enough for all of them).

    A step is :meth:`reserve`, then :meth:`append` (or :meth:`append_latent`) and the attention of every layer, then
    :meth:`advance`.  Positions that no page was reserved for are refused."""

    # New tokens per sequence that attend on the paged kernels; longer prompts read the cache back and use dense attention,
    # causal on an empty cache and with a mask behind earlier tokens.  Measured both ways for 1 to 64 sequences of 0 to 32000 cached
    # tokens, 8 to 128 new ones, three head layouts, windows, 8-bit and latent rows.  Behind cached tokens the pages are ahead up to
    # 128 new ones: 8 x 4000, 32 heads on 8, 16 new tokens 60 us and 236 dense, 128 tokens 338 and 436; 32 x 2000 683 and 781; at the
    # least 64 x 200, 329 and 328; with a window of 512, 8 x 4000, 100 and 459; a latent layer of 128 heads, 4 x 4000, 64 tokens, 0.62
    # and 4.7 ms.  On an empty cache 64 sequences of 16 tokens take 21 and 46 us, of 32 tokens 36 and 45, of 64 tokens 68 and 49.
    first_tokens, more_tokens = 16, 128

    def __init__(self, layers: int, heads: int, dim: int, batch: int, max_length: int, *, page: int = 64, e4m3: bool = False,
                 latent: bool = False, num_pages: Optional[int] = None, dtype: torch.dtype = torch.bfloat16, device="cpu") -> None:
        if min(layers, heads, dim, batch, max_length, page) < 1:
            raise ValueError("PagedKVCache: layers, heads, dim, batch, max_length and page must be positive")
        if latent and heads != 1:
            raise ValueError("PagedKVCache: a latent cache has one row per position")
        self.page, self.e4m3, self.latent, self.dtype, self.batch = page, e4m3, latent, dtype, batch
        self.max_length = max_length
        width = -(-max_length // page)
        self.num_pages = batch * width if num_pages is None else num_pages
        kind = torch.float8_e4m3fn if e4m3 else dtype

        def pages():
            return [torch.empty(self.num_pages, heads, page, dim, dtype=kind, device=device) for _ in range(layers)]

        def scales():
            return [torch.empty(self.num_pages, heads, page, device=device) if e4m3 else None for _ in range(layers)]

        self.k_pages, self.k_scale = pages(), scales()
        self.v_pages, self.v_scale = ([None] * layers, [None] * layers) if latent else (pages(), scales())
        self.page_table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self.starts = torch.zeros(batch, dtype=torch.int32, device=device)  # tokens cached so far, on the device
        self.lengths: List[int] = [0] * batch  # the same on the host
        self._held: List[List[int]] = [[] for _ in range(batch)]
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._room = 0  # positions that every sequence has pages for, behind its cached ones

    @classmethod
    def for_model(cls, cfg: ArchConfig, batch: int, max_length: int, **kw) -> "PagedKVCache":
        """A cache that fits a native model's config."""
        if cfg.get("kv_lora_rank") and cfg.get("qk_rope_head_dim"):
            return cls(cfg["num_hidden_layers"], 1, cfg["kv_lora_rank"] + cfg["qk_rope_head_dim"], batch, max_length, latent=True, **kw)
        heads = cfg.get("num_key_value_heads") or cfg["num_attention_heads"]
        return cls(cfg["num_hidden_layers"], heads, cfg.head_dim_, batch, max_length, **kw)

    # -- pages ------------------------------------------------------------------------------------
    def reserve(self, tokens: int) -> None:
        """Makes room for ``tokens`` more positions of every sequence."""
        need = [-(-(n + tokens) // self.page) - len(held) for n, held in zip(self.lengths, self._held)]
        if max(self.lengths) + tokens > self.max_length:
            raise ValueError(f"PagedKVCache: {max(self.lengths)} + {tokens} positions, but max_length is {self.max_length}")
        if sum(max(0, n) for n in need) > len(self._free):
            raise RuntimeError(f"PagedKVCache: {sum(max(0, n) for n in need)} pages needed, {len(self._free)} left of {self.num_pages}")
        grew = False
        for held, n in zip(self._held, need):
            for _ in range(n):
                held.append(self._free.pop())
                grew = True
        if grew:
            self._upload()

    def _check_room(self, tokens: int) -> None:
        if tokens > self._room:
            raise ValueError(f"PagedKVCache: {tokens} new positions, but some sequence has pages for {self._room} only; reserve them first")

    def advance(self, tokens: int) -> None:
        """The last ``tokens`` written positions of every sequence belong to it from now on (after all layers wrote them)."""
        self._check_room(tokens)
        self._room -= tokens
        self.lengths = [n + tokens for n in self.lengths]
        self.starts += tokens

    def release(self, sequence: int) -> None:
        """Forgets one sequence and gives its pages back."""
        self._free.extend(reversed(self._held[sequence]))
        self._held[sequence] = []
        self.lengths[sequence] = 0
        self.starts[sequence] = 0
        self._upload()

    def _upload(self) -> None:
        width = self.page_table.shape[1]
        rows = [held + [-1] * (width - len(held)) for held in self._held]
        self.page_table.copy_(torch.tensor(rows, dtype=torch.int32))
        self._room = min(min(len(held) * self.page, self.max_length) - n for held, n in zip(self._held, self.lengths))

    def positions(self, tokens: int) -> torch.Tensor:
        """Position ids ``[batch, tokens]`` of the next tokens."""
        return self.starts.long().unsqueeze(1) + torch.arange(tokens, device=self.starts.device)

    def on_pages(self, tokens: int) -> bool:
        """Whether ``tokens`` new tokens per sequence attend on the paged kernels."""
        return tokens <= (self.more_tokens if any(self.lengths) else self.first_tokens)

    # -- one layer --------------------------------------------------------------------------------
    def append(self, layer: int, q, k, v, cos, sin) -> torch.Tensor:
        """Rotates the new tokens' queries and keys, stores keys and values, returns the queries."""
        self._check_room(q.shape[1])
        return ops.paged_kv_append(q, k, v, cos, sin, self.k_pages[layer], self.v_pages[layer], self.page_table, self.starts, None,
                                   self.k_scale[layer], self.v_scale[layer])

    def append_latent(self, layer: int, q_pe, kv_a, norm_weight, eps: float, cos, sin) -> torch.Tensor:
        self._check_room(q_pe.shape[1])
        return ops.paged_latent_append(q_pe, kv_a, norm_weight, eps, cos, sin, self.k_pages[layer], self.page_table, self.starts, None,
                                       self.k_scale[layer])

    def attend(self, layer: int, q, scale: Optional[float] = None, window: Optional[int] = None, attn_impl: str = "sdpa") -> torch.Tensor:
        """Attention of the new tokens (already appended) over their sequences."""
        if self.on_pages(q.shape[1]):
            return ops.paged_attention(q, self.k_pages[layer], self.v_pages[layer], self.page_table, self.starts, None,
                                       self.k_scale[layer], self.v_scale[layer], scale, window)
        k, v = self.read(layer, q.shape[1], q.dtype)
        return self.prompt_attention(q, k, v, scale, window, attn_impl)

    def attend_latent(self, layer: int, q_latent, q_pe, scale: float) -> torch.Tensor:
        return ops.paged_latent_attention(q_latent, q_pe, self.k_pages[layer], self.page_table, self.starts, None, self.k_scale[layer],
                                          scale)

    def read(self, layer: int, new: int, dtype: torch.dtype) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """Everything cached so far and the ``new`` tokens just appended, ``[batch, longest, heads, dim]``."""
        return ops.paged_kv_read(self.k_pages[layer], self.v_pages[layer], self.page_table, self.starts + new, max(self.lengths) + new,
                                 self.k_scale[layer], self.v_scale[layer], dtype)

    def prompt_attention(self, q, k, v, scale: Optional[float], window: Optional[int] = None, attn_impl: str = "sdpa") -> torch.Tensor:
        """Dense attention of a prompt over keys and values that were read back."""
        S, L = q.shape[1], k.shape[1]
        if not any(self.lengths):
            return ops.attention(q, k, v, None, None, True, attn_impl, scale=scale, window=window)
        mine = self.positions(S).unsqueeze(-1)
        at = torch.arange(L, device=q.device)
        mask = at <= mine
        if window is not None:
            mask = mask & (at > mine - window)
        o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), attn_mask=mask.unsqueeze(1),
                                           scale=scale, enable_gqa=q.shape[2] != k.shape[2])
        return o.transpose(1, 2)
