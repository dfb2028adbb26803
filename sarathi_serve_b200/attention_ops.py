"""Attention of a step's new tokens over the paged KV cache (layout [pages, 2, page_size, kv_heads, head_dim]): prompt chunks
and single decoded tokens in one call, as the reference runs them through flashinfer's paged prefill wrapper
(sarathi/model_executor/attention/flashinfer_attention_wrapper.py:240-299).

``AttentionPlan`` is made once for a model shape and updated once a step -- on the GPU, without reading anything back, so a
step can be captured into a CUDA graph and replayed with other lengths; ``paged_attention`` is then called by every layer."""
from __future__ import annotations

import ctypes
from typing import List, Optional

import torch

from . import _native as N
from . import dense_ops
from .kv_cache_ops import BatchLayout, _int32


class AttentionPlan:
    """Division of a step's attention over the GPU, with the workspace its calls need.

    ``num_heads`` / ``num_kv_heads``: of this rank; ``window``: a token sees itself and the ``window - 1`` tokens before it (0:
    all of them).  ``max_requests`` and ``max_tokens`` bound the steps the plan is updated with.  A plan serves one step at a
    time: a call on another stream than the one before waits for that one, and the graphs that captured such calls belong on one
    stream (or ordered by events): replays that overlap give wrong numbers.  A graph keeps reading the ``kv_indices`` that the plan had
    when it was captured: write later steps' layouts to the same arrays (``batch_layout(..., out=)``), on the stream that reads them or
    ordered with it, as that call is none of the plan's."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int, dtype: torch.dtype, max_requests: int,
                 max_tokens: int, window: int = 0, device: Optional[torch.device] = None):
        if dtype not in N._DTYPE_ID:
            raise RuntimeError(f"AttentionPlan: unsupported dtype {dtype}")
        window = min(int(window or 0), N.INT_MAX)  # (no request is that long)
        self.shape = N.AttentionShape(*[N.int32(n, v, "AttentionPlan") for n, v in (
            ("num_heads", num_heads), ("num_kv_heads", num_kv_heads), ("head_dim", head_dim), ("page_size", page_size),
            ("dtype", N._DTYPE_ID[dtype]), ("window", window), ("max_requests", max_requests), ("max_tokens", max_tokens))])
        self._shape = ctypes.byref(self.shape)
        lib = N.lib()
        plan_bytes = lib.sb200_attention_plan_bytes(self._shape)
        if plan_bytes < 0:
            raise RuntimeError(lib.sb200_last_error().decode("utf-8", "replace"))
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.dtype = dtype
        self.num_heads, self.num_kv_heads, self.head_dim, self.page_size = num_heads, num_kv_heads, head_dim, page_size
        self.max_requests, self.max_tokens, self.window = max_requests, max_tokens, window
        self.buffer = torch.empty(plan_bytes, dtype=torch.uint8, device=device)
        self.workspace = torch.empty(lib.sb200_attention_workspace_bytes(self._shape), dtype=torch.uint8, device=device)
        self.kv_indices: Optional[torch.Tensor] = None
        self.beside: List[torch.Tensor] = []  # what else the plan's user reads on its streams: kept from reuse like the plan's own
        # the stream of the last call; so far the one that the buffers belong to
        self._stream = torch.cuda.current_stream(self.buffer.device)
        self._stream_ptr: int = self._stream.cuda_stream
        self._streams = {self._stream_ptr}  # those that the plan's own memory is kept for

    def stream(self) -> int:
        """The current stream, behind whatever the plan's calls have queued on the one they used last.  (A kernel that read a plan
        that is still being written would follow numbers that mean nothing.)  Not while a graph is captured: its replays are the
        caller's to order."""
        here = N.stream_ptr()
        if here != self._stream_ptr and not torch.cuda.is_current_stream_capturing():
            now = torch.cuda.current_stream()
            now.wait_stream(self._stream)
            if here not in self._streams:
                self._streams.add(here)
                for t in (self.buffer, self.workspace, *self.beside):
                    t.record_stream(now)
            if self.kv_indices is not None:
                self.kv_indices.record_stream(now)
            self._stream, self._stream_ptr = now, here
        return here

    def update(self, layout: Optional[BatchLayout] = None, *, qo_indptr: Optional[torch.Tensor] = None,
               kv_lens: Optional[torch.Tensor] = None, kv_indptr: Optional[torch.Tensor] = None,
               kv_indices: Optional[torch.Tensor] = None) -> "AttentionPlan":
        """Plan the step of ``layout`` (or of the four arrays given by name).  The plan keeps ``kv_indices`` and reads it in
        every ``paged_attention`` of the step; the others are read here only.  A layout that was made on another stream must be
        waited for there, as any tensor."""
        if layout is not None:
            qo_indptr, kv_lens, kv_indptr, kv_indices = layout[:4]
        if qo_indptr is None or kv_lens is None or kv_indptr is None or kv_indices is None:
            raise RuntimeError("AttentionPlan.update: needs a layout, or qo_indptr, kv_lens, kv_indptr and kv_indices")
        N.require_current(qo_indptr, kv_lens, kv_indptr, kv_indices, self.buffer)
        n = kv_lens.numel()
        for name, t, k in (("kv_lens", kv_lens, n), ("qo_indptr", qo_indptr, n + 1), ("kv_indptr", kv_indptr, n + 1),
                           ("kv_indices", kv_indices, -1)):
            _int32(name, t, k, "AttentionPlan.update")
        N.check(N.lib().sb200_attention_plan(self.buffer.data_ptr(), self.buffer.numel(), self._shape, qo_indptr.data_ptr(),
                                             kv_lens.data_ptr(), kv_indptr.data_ptr(), n, kv_indices.numel(), self.stream()),
                "attention_plan")
        if kv_indices is not self.kv_indices:
            # The plan lets go of it at some later update, when this stream may still be reading it.
            if not torch.cuda.is_current_stream_capturing():
                kv_indices.record_stream(self._stream)
            self.kv_indices = kv_indices
        return self


def paged_attention(q: torch.Tensor, paged_kv_cache: torch.Tensor, plan: AttentionPlan, scale: float,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = softmax(scale q[t] K^T) V per head, over the cached keys up to token t's position; this step's keys and values
    have been appended before.  q: [tokens, heads * head_dim] (or [tokens, heads, head_dim]); its rows may be a strided view of
    the fused qkv buffer.  Rows that belong to no request are zero in a result that is allocated here (-inf in ``lse``); in an
    ``out`` that is given they, and their ``lse``, are left as they were.  ``out`` may be strided like q, but must not overlap q or
    the cache.  ``lse``: optional fp32 [tokens, heads], the natural logarithm of the softmax denominators; it must not overlap any of
    the three."""
    N.require_current(q, paged_kv_cache, out, lse, plan.buffer)
    if plan.kv_indices is None:
        raise RuntimeError("paged_attention: the plan has not been updated with a step")
    heads, hd, dtype = plan.num_heads, plan.head_dim, plan.dtype
    T = q.shape[0]
    q2 = q.view(T, heads * hd) if q.dim() == 3 and q.shape[1:] == (heads, hd) else q
    if q2.dim() != 2 or q2.shape[1] != heads * hd or q2.stride(1) != 1:
        raise RuntimeError(f"paged_attention: q must be [tokens, {heads * hd}] with unit inner stride")
    if (paged_kv_cache.dim() != 5 or paged_kv_cache.shape[1:] != (2, plan.page_size, plan.num_kv_heads, hd)
            or not paged_kv_cache.is_contiguous()):
        raise RuntimeError(f"paged_attention: the cache must be a contiguous [pages, 2, {plan.page_size}, {plan.num_kv_heads}, {hd}] tensor")
    if q2.dtype != dtype or paged_kv_cache.dtype != dtype:
        raise RuntimeError("paged_attention: q and the cache must have the plan's dtype")
    clear = out is None
    if out is None:
        out = torch.empty(T, heads * hd, dtype=dtype, device=q.device)
    elif out.shape != (T, heads * hd) or out.dtype != dtype or out.stride(1) != 1:
        raise RuntimeError(f"paged_attention: out must be [tokens, {heads * hd}] of the plan's dtype with unit inner stride")
    if lse is not None and (lse.shape != (T, heads) or lse.dtype != torch.float32 or not lse.is_contiguous()):
        raise RuntimeError(f"paged_attention: lse must be a contiguous float32 tensor [tokens, {heads}]")
    kv = plan.kv_indices
    row = heads * hd
    N.check(N.lib().sb200_paged_attention(out.data_ptr(), out.stride(0) if T > 1 else row, N.ptr(lse), q2.data_ptr(),
                                          q2.stride(0) if T > 1 else row, T, paged_kv_cache.data_ptr(), paged_kv_cache.shape[0],
                                          plan.buffer.data_ptr(), plan._shape, kv.data_ptr(), kv.numel(), scale, 1 if clear else 0,
                                          plan.workspace.data_ptr(), plan.workspace.numel(),
                                          dense_ops.status_word(q.device).data_ptr(), plan.stream()), "paged_attention")
    return out
