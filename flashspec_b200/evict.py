"""Eviction from the paged INT8 cache by accumulated attention weight.

``paged_quant_attention_weights_cuda`` adds up, step by step, the attention that every
cached token receives; ``evict_tokens_cuda`` cuts requests down to a budget of tokens,
keeping the heaviest, the most recent and the first ones of every kv head, and packs them
into the request's first pages.  ``PagedKVAllocator`` (``track_weights=True``,
``evict_batch``) does the bookkeeping: it frees the pages that fall empty.  The reference
has no counterpart.

Keys keep whatever position encoding they were stored with; positions in the cut cache
number the kept tokens.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from .attention import _check_weights, _i64, _seq_cap
from .quant import device_guard, require_cuda, status_word, stream_of


def evict_tokens_cuda(cache, weights: torch.Tensor, budget: int, *, recent: int, sinks: int = 0,
                      weights_out: Optional[torch.Tensor] = None,
                      device_status: Optional[torch.Tensor] = None):
    """Cut every request of ``cache`` (a PagedKVCache) with more than ``budget`` tokens down
    to ``budget``: per kv head the first ``sinks`` and the last ``recent`` tokens and, of
    those between, the budget - sinks - recent with the largest ``weights`` (fp32 [P, Hkv,
    page] beside the pool; ties keep the earlier token).

    The pool is changed in place: the kept tokens move, in order, to the request's first
    pages (affine pages are requantized, as ``PagedKVAllocator.append_batch`` does; symmetric
    ones keep their codes), and their weights with them, or into ``weights_out`` (a tensor
    like ``weights`` that does not overlap it).  Positions behind the kept tokens get weight
    zero.  Requests within the budget keep their pages as they are.  Every page listed in
    the table must belong to one request: a page shared by requests cannot be changed in
    place.

    Returns (cut cache, kept): the cache with the same pool and table and the new lengths,
    and int32 [B, Hkv, budget], the kept tokens' former positions, -1 behind them.  No host
    synchronisation; everything runs on the current stream."""
    kq, vq = cache.k_quant, cache.v_quant
    require_cuda(kq.values, "the cache")
    device = kq.values.device
    if len(kq.original_shape) != 4 or tuple(kq.original_shape) != tuple(vq.original_shape):
        raise ValueError("cache.k_quant and cache.v_quant must be pools of one shape [pages, heads, page, head_dim]")
    sym = bool(getattr(kq, "symmetric", False))
    if sym != bool(getattr(vq, "symmetric", False)):
        raise ValueError("K and V must use the same quantization format")
    page, hkv, d = int(cache.block_size), int(kq.original_shape[1]), int(kq.original_shape[-1])
    if int(kq.block_size) != page or int(vq.block_size) != page or int(kq.original_shape[2]) != page:
        raise ValueError("eviction needs pages of one quantization block")
    pages = int(kq.values.shape[0])
    parts = [kq.values, vq.values, kq.scale, vq.scale] + ([] if sym else [kq.zero_point, vq.zero_point])
    if any(t.device != device for t in parts) or cache.block_table.device != device or cache.lengths.device != device:
        raise RuntimeError("the pool, block_table and lengths must be on one CUDA device")
    if not all(t.is_contiguous() for t in parts):
        raise ValueError("the pool is changed in place: its tensors must be contiguous")
    if any(t.dtype != want for t, want in zip(parts, (torch.int8,) * 2 + (torch.float32,) * 2 + (torch.int16,) * 2)):
        raise ValueError("a pool holds int8 values, fp32 scales and int16 zero points")
    _check_pool(parts, pages, hkv, page, d, sym)
    if kq.values.data_ptr() == vq.values.data_ptr():
        raise ValueError("K and V must be separate pools: both are changed in place")
    shape = (pages, hkv, page)
    _check_weights(weights, shape, device, "weights")
    out = weights if weights_out is None else weights_out
    if weights_out is not None:
        _check_weights(weights_out, shape, device, "weights_out")
        lo, hi = weights.data_ptr(), weights.data_ptr() + 4 * weights.numel()
        if out.data_ptr() != lo and out.data_ptr() < hi and out.data_ptr() + 4 * out.numel() > lo:
            raise ValueError("weights_out must be weights itself or not overlap it")
    budget, recent, sinks = int(budget), int(recent), int(sinks)
    if budget <= 0 or budget >= 1 << 30 or recent < 0 or sinks < 0 or recent + sinks > budget:
        raise ValueError("budget must be positive (below 2^30), recent and sinks not negative and together within the budget")
    table, lengths = _i64(cache.block_table), _i64(cache.lengths)
    if table.ndim != 2 or tuple(lengths.shape) != (table.shape[0],):
        raise ValueError("block_table must be [batch, columns] and lengths [batch]")
    b = int(table.shape[0])
    with device_guard(device):
        kept = torch.empty((b, hkv, budget), dtype=torch.int32, device=device)
        new_lengths = torch.empty(b, dtype=torch.int64, device=device)
        a = _lib.FsEvictArgs()
        a.kv_format = _lib.FS_KV_SYMMETRIC if sym else _lib.FS_KV_AFFINE_BLOCK
        a.batch, a.kv_heads, a.head_dim, a.page_size = b, hkv, d, page
        a.table_cols, a.max_seq_len = int(table.shape[1]), _seq_cap(int(cache.max_seq_len), page, int(table.shape[1]))
        a.budget, a.recent, a.sinks = budget, recent, sinks
        a.num_pages = pages
        a.block_table, a.lengths = table.data_ptr(), lengths.data_ptr()
        a.k_values, a.k_scale = kq.values.data_ptr(), kq.scale.data_ptr()
        a.v_values, a.v_scale = vq.values.data_ptr(), vq.scale.data_ptr()
        if not sym:
            a.k_zero, a.v_zero = kq.zero_point.data_ptr(), vq.zero_point.data_ptr()
        a.weights, a.weights_out = weights.data_ptr(), out.data_ptr()
        a.kept, a.new_lengths = kept.data_ptr(), new_lengths.data_ptr()
        a.device_status = status_word(device_status, device)
        lib, need = _lib.load(), C.c_size_t(0)
        _lib.check(lib.fs_evict_workspace_size(C.byref(a), C.byref(need)), "fs_evict_tokens")
        ws = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
        if ws is not None:
            a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
        _lib.check(lib.fs_evict_tokens(C.byref(a), stream_of(device)), "fs_evict_tokens")
    from .paged import PagedKVCache

    cut = PagedKVCache(kq, vq, cache.block_table, new_lengths, page, min(int(cache.max_seq_len), budget))
    return cut, kept


def _check_pool(parts, pages: int, hkv: int, page: int, d: int, sym: bool) -> None:
    """The kernels write to every part of the pool: raises unless K's and V's values, scales
    and zero points (in that order) have an entry for each page, head and token or block."""
    blocks = pages * hkv * (page if sym else 1)
    if any(t.numel() != pages * hkv * page * d for t in parts[:2]) or any(t.numel() != blocks for t in parts[2:]):
        raise ValueError("a pool's values, scales and zero points must all cover its pages, heads and tokens")
