"""Append of a step's keys and values to the paged KV cache (layout
[pages, 2, page_size, kv_heads, head_dim]), with the call signature of flashinfer's
``append_paged_kv_cache`` that the reference's attention wrapper uses
(sarathi/model_executor/attention/flashinfer_attention_wrapper.py:261-270).

``slots`` computes, once per step, the cache row of every token; ``append_paged_kv_cache`` copies
strided k / v views (no ``.contiguous()``) there.  ``dense_ops.linear_rotary(..., kv_cache=, kv_slots=)``
stores k and v from the qkv GEMM's epilogue instead, so that only ``slots`` remains as a launch.

``resize_block_tables`` and ``batch_layout`` make a step's block tables and index arrays on the GPU, from the lengths of
its requests: what the reference's block manager and its wrapper's ``begin_forward`` do in host loops.  Neither reads
anything back, so both can be captured into the CUDA graph of a step."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as N


def slots(batch_indices: torch.Tensor, positions: torch.Tensor, kv_indices: torch.Tensor, kv_indptr: torch.Tensor,
          page_size: int, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """int64 [n]: row of the cache (seen as [pages * 2 * page_size, kv_heads * head_dim]) that receives token i's key;
    -1 where ``batch_indices[i] < 0``."""
    N.require_cuda(batch_indices, positions, kv_indices, kv_indptr, out)
    for name, t in (("batch_indices", batch_indices), ("positions", positions), ("kv_indices", kv_indices),
                    ("kv_indptr", kv_indptr)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise RuntimeError(f"kv_cache_ops.slots: {name} must be a contiguous int32 tensor")
    n = batch_indices.numel()
    if positions.numel() != n:
        raise RuntimeError("kv_cache_ops.slots: batch_indices and positions differ in length")
    if out is None:
        out = torch.empty(n, dtype=torch.int64, device=batch_indices.device)
    N.check(N.lib().sb200_kv_cache_slots(N.ptr(out), N.ptr(batch_indices), N.ptr(positions), N.ptr(kv_indices),
                                         N.ptr(kv_indptr), n, N.int32("page_size", page_size, "kv_cache_ops.slots"), N.stream_ptr()), "kv_cache_slots")
    return out


def append_rows(paged_kv_cache: torch.Tensor, key: torch.Tensor, value: torch.Tensor, kv_slots: torch.Tensor) -> None:
    """key / value: [n, kv_heads * head_dim] (or [n, kv_heads, head_dim]), rows may be strided views of the
    fused qkv buffer; ``kv_slots`` from ``slots``."""
    N.require_cuda(paged_kv_cache, key, value, kv_slots)
    if paged_kv_cache.dim() != 5 or paged_kv_cache.shape[1] != 2 or not paged_kv_cache.is_contiguous():
        raise RuntimeError("append_rows: the cache must be a contiguous [pages, 2, page_size, kv_heads, head_dim] tensor")
    _, _, page, nkv, hd = paged_kv_cache.shape
    n = kv_slots.numel()
    k2 = key.reshape(n, -1) if key.dim() == 3 and key.is_contiguous() else key.view(n, -1) if key.dim() == 3 else key
    v2 = value.reshape(n, -1) if value.dim() == 3 and value.is_contiguous() else value.view(n, -1) if value.dim() == 3 else value
    for name, t in (("key", k2), ("value", v2)):
        if t.dim() != 2 or t.shape != (n, nkv * hd) or t.stride(1) != 1 or t.dtype != paged_kv_cache.dtype:
            raise RuntimeError(f"append_rows: {name} must be [n, kv_heads * head_dim] with unit inner stride and the cache's dtype")
    if kv_slots.dtype != torch.int64 or not kv_slots.is_contiguous():
        raise RuntimeError("append_rows: kv_slots must be a contiguous int64 tensor")
    N.check(N.lib().sb200_kv_cache_append(N.ptr(paged_kv_cache), N.ptr(k2), k2.stride(0), N.ptr(v2), v2.stride(0),
                                          N.ptr(kv_slots), n, nkv, hd, page, N.dtype_id(k2), N.stream_ptr()),
            "kv_cache_append")


def append_paged_kv_cache(append_key: torch.Tensor, append_value: torch.Tensor, batch_indices: torch.Tensor,
                          positions: torch.Tensor, paged_kv_cache: torch.Tensor, kv_indices: torch.Tensor,
                          kv_indptr: torch.Tensor, kv_last_page_len: Optional[torch.Tensor] = None,
                          kv_layout: str = "NHD") -> None:
    """Drop-in for ``flashinfer.append_paged_kv_cache`` with a single 5-D NHD cache tensor (what the reference
    allocates).  ``kv_last_page_len`` is accepted and unused (flashinfer's kernel does not read it either: the
    slot follows from the position)."""
    if kv_layout != "NHD":
        raise RuntimeError("append_paged_kv_cache: only the NHD layout of the reference's cache is supported")
    s = slots(batch_indices, positions, kv_indices, kv_indptr, paged_kv_cache.shape[2])
    append_rows(paged_kv_cache, append_key, append_value, s)


def _int32(name: str, t: torch.Tensor, n: int, what: str) -> None:
    if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous() or (n >= 0 and t.numel() != n):
        raise RuntimeError(f"{what}: {name} must be a contiguous int32 tensor" + (f" of {n} elements" if n >= 0 else ""))


def _tables(block_tables: torch.Tensor, n: int, what: str) -> None:
    if block_tables.dtype is not torch.int32 or block_tables.dim() != 2 or block_tables.size(0) != n:
        raise RuntimeError(f"{what}: block_tables must be an int32 tensor [{n}, blocks]")
    width = block_tables.size(1)
    if (width > 1 and block_tables.stride(1) != 1) or (n > 1 and block_tables.stride(0) < width):
        raise RuntimeError(f"{what}: the rows of block_tables must have unit inner stride and must not overlap")


def _table_stride(block_tables: torch.Tensor) -> int:
    return block_tables.stride(0) if block_tables.shape[0] > 1 else block_tables.shape[1]


def resize_block_tables(block_tables: torch.Tensor, num_blocks: torch.Tensor, seq_lens: torch.Tensor, free_blocks: torch.Tensor,
                        num_free: torch.Tensor, page_size: int, granted: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Make the block tables fit the requests' lengths, in place: afterwards request r owns ceil(seq_lens[r] / page_size)
    pages, entries [0, num_blocks[r]) of ``block_tables`` [n, blocks].  A request that shrinks (``seq_lens[r] = 0``: it has
    finished) pushes its last pages on the stack ``free_blocks[:num_free]``; then requests that grow pop theirs from its top,
    in request order.  Returns ``granted`` int32 [n]: 0 where the stack (or the table's width) did not suffice and the request
    was left as it was -- from the first such request on, none that needs pages gets any, unless it was its own table that was
    too narrow.  A negative length leaves a request alone.  All tensors int32 on the GPU, none overlapping another; ``num_free`` has one element."""
    what = "resize_block_tables"
    N.require_current(block_tables, num_blocks, seq_lens, free_blocks, num_free, granted)
    n = num_blocks.numel()
    _tables(block_tables, n, what)
    for name, t, k in (("num_blocks", num_blocks, n), ("seq_lens", seq_lens, n), ("free_blocks", free_blocks, -1),
                       ("num_free", num_free, 1)):
        _int32(name, t, k, what)
    if granted is None:
        granted = torch.empty(n, dtype=torch.int32, device=num_blocks.device)
    else:
        _int32("granted", granted, n, what)
    N.check(N.lib().sb200_resize_block_tables(N.ptr(block_tables), _table_stride(block_tables), N.ptr(num_blocks), N.ptr(seq_lens),
                                              N.ptr(free_blocks), N.ptr(num_free), N.ptr(granted), n, block_tables.shape[1],
                                              free_blocks.numel(), N.int32("page_size", page_size, what), N.stream_ptr()), what)
    return granted


class _BatchArrays(NamedTuple):
    qo_indptr: torch.Tensor      # int32 [n + 1]
    kv_lens: torch.Tensor        # int32 [n]
    kv_indptr: torch.Tensor      # int32 [n + 1]
    kv_indices: torch.Tensor     # int32 [n * blocks]
    last_page_len: torch.Tensor  # int32 [n]
    batch_indices: torch.Tensor  # int32 [num_tokens]
    positions: torch.Tensor      # int64 [num_tokens]
    kv_slots: torch.Tensor       # int64 [num_tokens]


class BatchLayout(_BatchArrays):
    """Index arrays of a step (see ``batch_layout``).  ``_for``: the sizes, device, addresses and lengths that ``batch_layout`` made or
    checked them for, so that a step that writes the same arrays again need not look at eight types, shapes and strides."""
    _for = None


def batch_layout(query_lens: torch.Tensor, context_lens: torch.Tensor, block_tables: torch.Tensor, page_size: int, num_pages: int,
                 num_tokens: int, out: Optional[BatchLayout] = None) -> BatchLayout:
    """Index arrays of a step in which request r adds ``query_lens[r]`` tokens to the ``context_lens[r]`` it has in the cache,
    all new tokens one after the other in a batch padded to ``num_tokens`` rows: row offsets (``qo_indptr``), lengths
    (``kv_lens``), page lists in the form of flashinfer's plan (``kv_indptr``, ``kv_indices``, ``last_page_len``; -1 behind the
    last page), and for every row its request (-1: padding), position and cache slot (-1: padding, or a page outside
    ``[0, num_pages)``).  ``positions`` goes to the rotary embedding, ``kv_slots`` to the append, everything to
    ``attention_ops.AttentionPlan.update``.

    Negative lengths count as zero.  A context is cut to what its block table has room for, and the new tokens to what is then
    left of it and of ``num_tokens``.  ``out``: the result of an earlier call of the same sizes, written again (buffers of a CUDA
    graph); its arrays must not be inputs too (``context_lens=out.kv_lens.clone()`` for the step after)."""
    what = "batch_layout"
    n = query_lens.numel()
    N.require_current(query_lens, context_lens, block_tables)
    _int32("query_lens", query_lens, n, what)
    _int32("context_lens", context_lens, n, what)
    _tables(block_tables, n, what)
    T, width, dev = int(num_tokens), block_tables.shape[1], query_lens.device
    if T < 0:
        raise RuntimeError(f"{what}: num_tokens is negative")
    made = out is None
    if made:
        # one allocation each for the two types; the parts of either one after the other
        parts = [n + 1, n, n + 1, n * width, n, T]
        ints = torch.empty(sum(parts), dtype=torch.int32, device=dev)
        longs = torch.empty(2 * T, dtype=torch.int64, device=dev)
        # ("unsafe": without the bookkeeping of autograd for views, which integers have no use for)
        out = BatchLayout(*torch.unsafe_split_with_sizes(ints, parts), *torch.unsafe_split_with_sizes(longs, [T, T]))
    at, lengths = [*map(torch.Tensor.data_ptr, out)], [*map(torch.Tensor.numel, out)]
    this = (n, width, T, dev, at, lengths)
    if not made and out._for != this:
        N.require_current(*out)
        for name, t, k in zip(BatchLayout._fields, out, (n + 1, n, n + 1, -1, n, T)):
            _int32("out." + name, t, k, what)
        if out.kv_indices.numel() < n * width:
            raise RuntimeError(f"{what}: out.kv_indices must hold {n * width} entries")
        for t in out[6:]:
            if t.dtype != torch.int64 or t.shape != (T,) or not t.is_contiguous():
                raise RuntimeError(f"{what}: out.positions and out.kv_slots must be contiguous int64 tensors of {T} elements")
    out._for = this
    qo, kv, indptr, indices, last, req, pos, slot = at
    N.check(N.lib().sb200_batch_layout(query_lens.data_ptr(), context_lens.data_ptr(), block_tables.data_ptr(), _table_stride(block_tables),
                                       n, width, N.int32("page_size", page_size, what), int(num_pages), T, qo, kv, indptr, indices,
                                       lengths[3], last, req, pos, slot, N.stream_ptr()), what)
    return out
