"""Paged key/value cache and the dense decoder over it, for prompts of different lengths.

``PagedDenseStack`` is :class:`~moeinfra_b200.engine.dense.DenseStack` with the static cache
``[B, kv_heads, max_len, head_dim]`` replaced by pages that sequences take as they need them, and
the library attention by this package's kernels: per layer one ``rope_append`` (rotation of q and
k, append of k and v) and one ``prompt_attention`` (prompts, packed without padding) or
``paged_attention`` (a decode step, each sequence at its own length).  The reference has neither
(one sequence over a growing ``DynamicCache``, ``engine/engine.py:326-378``).

Rotation here is fp32 arithmetic on an fp32 table, rounded once; the static path rotates in fp16
as Hugging Face's modules do, so the two paths' logits differ by fp16 rounding.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from moeinfra_b200 import kernels
from moeinfra_b200.engine.dense import DenseStack, rms_norm


class PagedKVCache:
    """Pages of all layers, a block table for ``max_batch`` sequences, and the free list (host)."""

    def __init__(self, num_layers: int, num_pages: int, kv_heads: int, page_size: int,
                 head_dim: int, max_batch: int, max_len: int, device, dtype=torch.float16) -> None:
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
        shape = (num_layers, num_pages, kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros_like(self.k_pages)
        self.page_size = page_size
        self.block_table = torch.full((max_batch, -(-max_len // page_size)), -1, dtype=torch.int32,
                                      device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._held: dict[int, list[int]] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, lengths: list[int]) -> None:
        """Give sequence b pages for ``lengths[b]`` positions (all or none; releases what it held)."""
        self.release()
        need = [-(-n // self.page_size) for n in lengths]
        rows, width = self.block_table.shape
        if len(need) > rows or any(n > width for n in need):
            raise ValueError(f"{len(need)} sequences of up to {max(lengths)} positions exceed the "
                             f"block table of {rows} x {width} pages")
        if sum(need) > len(self._free):
            raise RuntimeError(f"the paged cache has {len(self._free)} free pages, "
                               f"{sum(need)} are needed (engine.kv_pages)")
        table = torch.full((rows, width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            self._held[b] = [self._free.pop() for _ in range(n)]
            table[b, :n] = torch.tensor(self._held[b], dtype=torch.int32)
        self.block_table.copy_(table)

    def release(self) -> None:
        """Take every sequence's pages back."""
        for pages in self._held.values():
            self._free.extend(reversed(pages))
        self._held.clear()


class PagedDenseStack(DenseStack):
    """The dense decoder stack over a :class:`PagedKVCache`; head_dim 64 or 128, fp16 or bf16."""

    def __init__(self, *args, page_size: int = 64, num_pages: int | None = None, **kwargs) -> None:
        self._page_size, self._num_pages = page_size, num_pages
        super().__init__(*args, **kwargs)

    def _make_cache(self, angles: torch.Tensor) -> None:
        cfg = self.cfg
        if cfg.head_dim not in (64, 128):
            raise ValueError(f"the paged cache's kernels take head_dim 64 or 128, not {cfg.head_dim}")
        per_seq = -(-self.max_len // self._page_size) if self._page_size > 0 else 0
        pages = self.max_batch * per_seq if self._num_pages is None else self._num_pages
        self.cache = PagedKVCache(len(self.layers), pages, cfg.num_kv_heads, self._page_size,
                                  cfg.head_dim, self.max_batch, self.max_len, self.device, self.dtype)
        half = angles[:, :cfg.head_dim // 2]
        self.cos, self.sin = half.cos().contiguous(), half.sin().contiguous()
        # One workspace for the layers' attention calls, which follow one another.
        self._workspace = kernels.paged_attention_workspace(
            self.cache.block_table, self._page_size, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim)

    def _layers(self, h: torch.Tensor, attend) -> torch.Tensor:
        eps = self.cfg.rms_norm_eps
        for li, lay in enumerate(self.layers):
            qkv = F.linear(rms_norm(h, lay.in_norm, eps), lay.w_qkv)
            o = attend(li, qkv)
            h = h + F.linear(o.view(h.shape[0], -1), lay.w_o)
            y = self.moe[li].forward(rms_norm(h, lay.post_norm, eps))
            if self.layer_hook is not None:
                self.layer_hook(li, self.moe[li])
            h = h + y
        return h

    def _logits(self, h: torch.Tensor) -> torch.Tensor:
        return F.linear(rms_norm(h, self.final_norm, self.cfg.rms_norm_eps), self.lm_head)

    def prefill(self, prompts: list[torch.Tensor]) -> torch.Tensor:
        """Whole prompts, packed: each a 1-D tensor of ids; fp16 logits of their last positions.

        The cache must hold pages for them (``cache.reserve``).  ``prompt_lengths`` then is their
        lengths on the device, int32: the positions of the tokens that follow."""
        cfg = self.cfg
        lens = [int(p.numel()) for p in prompts]
        if not lens or min(lens) < 1 or max(lens) > self.max_len or len(lens) > self.max_batch:
            raise ValueError(f"{len(lens)} prompts of {lens} tokens: 1 to {self.max_batch} prompts "
                             f"of 1 to {self.max_len} tokens are served")
        ids = torch.cat([p.reshape(-1) for p in prompts]).to(device=self.device, dtype=torch.long)
        n = torch.tensor(lens)
        cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
        cu[1:] = n.cumsum(0)
        seq = torch.repeat_interleave(torch.arange(len(lens), dtype=torch.int32), n)
        pos = torch.arange(len(seq), dtype=torch.int32) - cu[seq.long()]
        last = (cu[1:] - 1).long().to(self.device)
        cu, seq, pos = (t.to(self.device) for t in (cu, seq, pos))
        self.prompt_lengths = cu.diff()
        H, KV, hd = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim
        table = self.cache.block_table

        def attend(li: int, qkv: torch.Tensor) -> torch.Tensor:
            k = qkv.new_empty((qkv.shape[0], KV, hd))
            q = kernels.rope_append(qkv, self.cos, self.sin, pos, table, self.cache.k_pages[li],
                                    self.cache.v_pages[li], H, seq_ids=seq, k_out=k)
            v = qkv.view(-1, H + 2 * KV, hd)[:, H + KV:]
            return kernels.prompt_attention(q, k, v, cu, max(lens), scale=self.scale,
                                            workspace=self._workspace)

        return self._logits(self._layers(F.embedding(ids, self.embed), attend)[last])

    def decode(self, ids: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """One token per sequence: ids [B, 1], its position in its sequence int32 [B]; logits."""
        cfg, B = self.cfg, ids.shape[0]
        table = self.cache.block_table[:B]
        lengths = positions + 1

        def attend(li: int, qkv: torch.Tensor) -> torch.Tensor:
            kp, vp = self.cache.k_pages[li], self.cache.v_pages[li]
            q = kernels.rope_append(qkv, self.cos, self.sin, positions, table, kp, vp, cfg.num_heads)
            return kernels.paged_attention(q, kp, vp, table, lengths, scale=self.scale,
                                           workspace=self._workspace)

        return self._logits(self._layers(F.embedding(ids[:, 0], self.embed), attend))

    def forward(self, ids, pos0=0, decode_pos=None):
        raise NotImplementedError("a paged stack is driven by prefill() and decode()")
