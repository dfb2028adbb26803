"""Attention backend of the decoder layers on this package's own kernels: what the reference's flashinfer wrapper is to its
models (sarathi/model_executor/attention/flashinfer_attention_wrapper.py: the paged caches :69-77, begin_forward,
forward :240-299, end_forward of base_attention_wrapper.py:50-79).

Between ``begin_forward`` and ``end_forward`` the layers call ``forward(q, k, v, layer_cache_idx, scale, layer_id)``.  A layer
that asks for ``fused_kv_append`` first stores this step's keys and values from its qkv projection; for one that does not,
``forward`` appends them."""
from __future__ import annotations

from typing import List, Optional

import torch

from . import _native as N
from . import attention_ops, kv_cache_ops


class PagedAttentionWrapper:
    """Paged caches of ``num_layers`` layers and the plan of the current step.

    Everything a step changes lies in buffers of fixed address, sized for ``max_requests`` requests of ``max_blocks`` pages and
    ``max_tokens`` rows: ``begin_forward`` fills them on the current stream (copies and two kernels), and whatever was captured with this
    wrapper -- ``graph_runner.LayerGraph``, ``model_runner.ModelGraphRunner`` -- can be replayed after it, for any step of as
    many rows.  One step at a time: replays and ``begin_forward`` belong on one stream."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, num_pages: int, num_layers: int,
                 dtype: torch.dtype, max_requests: int, max_tokens: int, max_blocks: int, window: int = 0,
                 device: Optional[torch.device] = None):
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.num_kv_heads, self.head_dim, self.page_size, self.num_pages = num_kv_heads, head_dim, page_size, num_pages
        self.max_requests, self.max_tokens, self.max_blocks = max_requests, max_tokens, max_blocks
        self.plan = attention_ops.AttentionPlan(num_heads, num_kv_heads, head_dim, page_size, dtype, max_requests, max_tokens,
                                                window=window, device=device)
        self.kv_caches: List[torch.Tensor] = [torch.zeros(num_pages, 2, page_size, num_kv_heads, head_dim, dtype=dtype, device=device)
                                              for _ in range(num_layers)]
        ints = dict(dtype=torch.int32, device=device)
        self.query_lens = torch.zeros(max_requests, **ints)
        self.context_lens = torch.zeros(max_requests, **ints)
        self.block_tables = torch.full((max_requests, max_blocks), -1, **ints)
        self.layout = kv_cache_ops.batch_layout(self.query_lens, self.context_lens, self.block_tables, page_size, num_pages, max_tokens)
        self.plan.update(self.layout)
        # (the layout's arrays are parts of two allocations)
        self.plan.beside = [self.query_lens, self.context_lens, self.block_tables, self.layout.qo_indptr, self.layout.positions,
                            *self.kv_caches]
        self.num_tokens = max_tokens
        self._appended: Optional[int] = None

    @property
    def positions(self) -> torch.Tensor:
        """int64 [max_tokens]: position of every row of the step (0 for padding)."""
        return self.layout.positions

    def begin_forward(self, query_lens: torch.Tensor, context_lens: torch.Tensor, block_tables: torch.Tensor,
                      num_tokens: int) -> None:
        """The next step: request r adds ``query_lens[r]`` tokens to the ``context_lens[r]`` it has in the cache, in pages
        ``block_tables[r]``, in a batch padded to ``num_tokens`` rows (of a graph: the rows it was captured with).  int32
        tensors, on the device or on the host, of at most ``max_requests`` requests and ``max_blocks`` pages each.  Nothing is
        synchronised: pinned host tensors are read when the stream gets there, so they keep their values until then.  A request
        whose length reaches behind its pages sees zeros there and stores nothing; tokens behind row ``num_tokens`` are no part
        of the step's results."""
        if not 0 <= num_tokens <= self.max_tokens:
            raise RuntimeError(f"begin_forward: {num_tokens} rows, made for at most {self.max_tokens}")
        n = query_lens.numel()
        if context_lens.numel() != n or block_tables.dim() != 2 or block_tables.shape[0] != n:
            raise RuntimeError("begin_forward: query_lens, context_lens and block_tables are of different lengths")
        if n > self.max_requests or block_tables.shape[1] > self.max_blocks:
            raise RuntimeError(f"begin_forward: made for at most {self.max_requests} requests of {self.max_blocks} pages, got "
                               f"{n} of {block_tables.shape[1]}")
        for t in (query_lens, context_lens, block_tables):
            if t.dtype != torch.int32:
                raise RuntimeError("begin_forward: query_lens, context_lens and block_tables must be int32")
        N.require_current(self.query_lens)
        self.plan.stream()
        self.query_lens[:n].copy_(query_lens.reshape(-1), non_blocking=True)
        self.context_lens[:n].copy_(context_lens.reshape(-1), non_blocking=True)
        width = block_tables.shape[1]
        self.block_tables[:n, :width].copy_(block_tables, non_blocking=True)
        if width < self.max_blocks:  # what the step before left there is no page of this one
            self.block_tables[:n, width:].fill_(-1)
        if n < self.max_requests:
            self.query_lens[n:].zero_()
            self.context_lens[n:].zero_()
        kv_cache_ops.batch_layout(self.query_lens, self.context_lens, self.block_tables, self.page_size, self.num_pages, self.max_tokens,
                                  out=self.layout)
        self.plan.update(self.layout)
        self.num_tokens = num_tokens
        self._appended = None

    def end_forward(self) -> None:
        self._appended = None

    def get_cache_block(self, layer_cache_idx: int) -> torch.Tensor:
        return self.kv_caches[layer_cache_idx]

    def fused_kv_append(self, layer_cache_idx: int):
        """(paged cache, slots) for the qkv projection's epilogue: the layer stores its own keys and values."""
        cache = self.kv_caches[layer_cache_idx]
        N.require_current(cache)
        self.plan.stream()
        self._appended = layer_cache_idx
        return cache, self.layout.kv_slots[:self.num_tokens]

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, layer_cache_idx: int, softmax_scale: float = 1.0,
                layer_id: Optional[int] = None) -> torch.Tensor:
        """[T, heads * head_dim] from the step's rotated queries and keys and its values (views of the fused qkv buffer)."""
        T = query.shape[0]
        if T > self.max_tokens:
            raise RuntimeError(f"PagedAttentionWrapper: {T} rows, made for at most {self.max_tokens}")
        cache = self.kv_caches[layer_cache_idx]
        N.require_current(query, key, value, cache)
        self.plan.stream()
        if self._appended != layer_cache_idx:
            kv_cache_ops.append_rows(cache, key, value, self.layout.kv_slots[:T])
        self._appended = None
        return attention_ops.paged_attention(query, cache, self.plan, softmax_scale)
