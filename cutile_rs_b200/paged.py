"""A paged key/value cache and the batches that use it: the containers behind ``launch.paged_*``.

The reference keeps one dense cache per sequence (cutile-kernels/src/kv_cache.rs); here many sequences share a pool of
pages.  Both classes only describe device memory that a ``torch.Tensor`` owns, so that a serving loop builds them once
and updates lengths, tables and rows in place.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .tensor import TensorError, dtype_name


def _strides(name: str, t: torch.Tensor):
    if t.stride(3) != 1:
        raise TensorError(f"the head vectors of {name} must be contiguous")
    return (ctypes.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2))


class PagedKvCache:
    """K and V pools [pages, kv_heads, page_size, D], of 16-bit elements, or of NVFP4 blocks: ``k`` and ``v`` uint8
    [.., D / 2] with two codes per byte (low nibble first) and ``k_scales``, ``v_scales`` uint8 or float8_e4m3fn
    [.., D / 16]; a value is code * scale * ``k_global`` (``v_global``).  Any strides: a pool kept as
    [pages, page_size, kv_heads, D] is passed permuted.  D is 64 or 128, page_size a power of two from 16."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None, k_global: float = 1.0, v_global: float = 1.0):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise TensorError("K and V pools must be [pages, kv_heads, page_size, D] of the same shape and type")
        if (k_scales is None) != (v_scales is None):
            raise TensorError("k_scales and v_scales are given together or not at all")
        self.tensors = (k, v, k_scales, v_scales)
        self.device = k.device
        self.num_pages, self.kv_heads, self.page_size, last = (int(s) for s in k.shape)
        fp4 = k_scales is not None
        self.head_dim = 2 * last if fp4 else last
        self.dtype: Optional[str] = None if fp4 else dtype_name(k.dtype)   # None: serves both 16-bit types
        c = _lib.PagedCacheC()
        if fp4:
            want = (self.num_pages, self.kv_heads, self.page_size, self.head_dim // 16)
            if k.dtype != torch.uint8:
                raise TensorError(f"NVFP4 pools are packed bytes (uint8), not {k.dtype}")
            for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
                if tuple(t.shape) != want or t.dtype not in (torch.uint8, torch.float8_e4m3fn):
                    raise TensorError(f"{name} must be uint8 or float8_e4m3fn {list(want)}")
            c.k_scales, c.v_scales = k_scales.data_ptr(), v_scales.data_ptr()
            c.k_scale_strides, c.v_scale_strides = _strides("k_scales", k_scales), _strides("v_scales", v_scales)
        elif self.dtype not in ("bf16", "f16"):
            raise TensorError(f"a cache holds bf16, f16 or NVFP4 blocks, not {k.dtype}")
        if any(t is not None and t.device != self.device for t in self.tensors):
            raise TensorError("the pools of a cache must be on one device")
        c.k, c.v = k.data_ptr(), v.data_ptr()
        c.k_strides, c.v_strides = _strides("k", k), _strides("v", v)
        c.k_global, c.v_global, c.format = float(k_global), float(v_global), int(fp4)
        c.num_pages, c.kv_heads, c.page_size, c.head_dim = self.num_pages, self.kv_heads, self.page_size, self.head_dim
        self._struct = c
        self.c = ctypes.addressof(c)      # what the C ABI takes


class PagedBatch:
    """The sequences of a call, int32 on the device: ``cu_q`` [batch + 1] (token rows of sequence b:
    [cu_q[b], cu_q[b + 1])), ``kv_lens`` [batch] (cached length, the new tokens included), ``block_table``
    [batch, max_pages].  ``max_q_len`` bounds the tokens of one sequence.  The contents are read when a kernel runs: they
    may be rewritten between calls and between replays of a captured graph.  Kernels are chosen by ``max_q_len`` and the
    table's width: bounds that fit the step (1 for decode steps, ``table[:, :pages_in_use]``) are faster than capacities."""

    def __init__(self, block_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, max_q_len: int):
        batch = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
        if block_table.dim() != 2 or batch < 0 or block_table.shape[0] != batch or tuple(cu_q.shape) != (batch + 1,):
            raise TensorError("expected block_table [batch, max_pages], cu_q [batch + 1], kv_lens [batch]")
        self.tensors = (block_table, cu_q, kv_lens)
        self.device = kv_lens.device
        if any(t.dtype != torch.int32 or t.device != self.device for t in self.tensors):
            raise TensorError("block_table, cu_q and kv_lens must be int32 on one device")
        if any(t.shape[-1] > 1 and t.stride(-1) != 1 for t in self.tensors):
            raise TensorError("block_table rows, cu_q and kv_lens must be contiguous")
        self.batch, self.max_pages, self.max_q_len = batch, int(block_table.shape[1]), int(max_q_len)
        c = _lib.PagedBatchC()
        c.block_table, c.block_table_pitch = block_table.data_ptr(), block_table.stride(0)
        c.cu_q, c.kv_lens = cu_q.data_ptr(), kv_lens.data_ptr()
        c.batch, c.max_pages, c.max_q_len = self.batch, self.max_pages, self.max_q_len
        self._struct = c
        self.c = ctypes.addressof(c)      # what the C ABI takes
