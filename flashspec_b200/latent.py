"""Latent cache and the two forms of attention over it.

A model with latent attention stores one shared vector a token instead of every head's keys
and values: a latent c (quantized here to INT8, one fp32 scale a token) and a rotary key
part r that all heads share.  ``LatentKVCache`` holds them in pages;

* ``LatentKVCache.append`` writes new tokens,
* ``latent_attention_cuda`` is the absorbed form for decoding: the queries are multiplied
  into the latent space by the caller (q_latent = q_nope W_uk of the head), the result comes
  back as a latent that the caller multiplies by W_uv;
* ``latent_prefill_attention_cuda`` is the expanded form for prompts, over every head's keys
  and values as the caller expanded them (``append(..., return_held=True)`` gives the latents
  that the cache stands for).

The reference has no counterpart.
"""

from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .attention import _i64, _seq_cap
from .quant import device_guard, require_cuda, status_word, stream_of

LATENT_DIMS = (128, 256, 512)
ROPE_DIMS = (32, 64)
LATENT_PAGES = (16, 32, 64, 128)


@dataclass(frozen=True)
class LatentKVCache:
    """Paged latent cache: ``values`` int8 [P, page, dc], ``scale`` fp32 [P, page] (not
    negative), ``ropes`` fp16 / bf16 [P, page, dr], ``block_table`` int64 [B, cols] (-1 = unallocated),
    ``lengths`` int64 [B], ``max_seq_len`` no less than any length.  dc 128, 256 or 512, dr 32
    or 64, page 16, 32, 64 or 128."""

    values: torch.Tensor
    scale: torch.Tensor
    ropes: torch.Tensor
    block_table: torch.Tensor
    lengths: torch.Tensor
    max_seq_len: int

    @property
    def batch_size(self) -> int:
        return int(self.block_table.shape[0])

    @property
    def block_size(self) -> int:
        return int(self.values.shape[1])

    @property
    def latent_dim(self) -> int:
        return int(self.values.shape[2])

    @property
    def rope_dim(self) -> int:
        return int(self.ropes.shape[2])

    @classmethod
    def empty(cls, batch: int, max_tokens: int, latent_dim: int = 512, rope_dim: int = 64, block_size: int = 64, *,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "LatentKVCache":
        """An empty cache with pages for ``max_tokens`` tokens of each request."""
        if batch <= 0 or max_tokens <= 0 or block_size <= 0:
            raise ValueError("batch, max_tokens and block_size must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("LatentKVCache lives on a CUDA device")
        cols = (int(max_tokens) + block_size - 1) // block_size
        pages = batch * cols
        cache = cls(torch.zeros((pages, block_size, latent_dim), dtype=torch.int8, device=device),
                    torch.zeros((pages, block_size), dtype=torch.float32, device=device),
                    torch.zeros((pages, block_size, rope_dim), dtype=dtype, device=device),
                    torch.arange(pages, dtype=torch.int64, device=device).view(batch, cols),
                    torch.zeros(batch, dtype=torch.int64, device=device), 0)
        _check_cache(cache)
        return cache

    def append(self, latent: torch.Tensor, rope: torch.Tensor, counts: Optional[torch.Tensor] = None, *,
               return_held: bool = False, device_status: Optional[torch.Tensor] = None):
        """Write new tokens behind each request's length: latent [B, T, dc] and rope [B, T, dr]
        in the cache's dtype (any strides with a dense last axis); ``counts`` int64 [B] of them
        for each request, all T where it is None.  Returns the cache with the new lengths (the
        pool is shared and changed in place).  The table must hold pages for them: a token
        without one is dropped, its position stays behind a hole, and FS_DEV_BAD_PAGE is set in
        ``device_status``; max_seq_len grows by T, at most to the table's end.

        ``return_held`` also returns the values that the cache now stands for, [B, T, dc] in
        the cache's dtype (zeros behind a request's count): what a prompt's expanded keys and
        values should be made of to agree with later steps."""
        _check_cache(self)
        pages, page, dc = self.values.shape
        dr = self.ropes.shape[2]
        device, dtype = self.values.device, self.ropes.dtype
        if latent.ndim != 3 or rope.ndim != 3:
            raise ValueError("latent and rope must be [batch, tokens, dim]")
        b, t, _ = latent.shape
        if b != self.block_table.shape[0] or t <= 0 or latent.shape[2] != dc or rope.shape != (b, t, dr):
            raise ValueError("latent must be [batch, tokens > 0, latent_dim] and rope [batch, tokens, rope_dim]")
        if latent.dtype != dtype or rope.dtype != dtype:
            raise ValueError("latent and rope must have the cache's dtype")
        if latent.device != device or rope.device != device:
            raise RuntimeError("latent and rope must be on the cache's CUDA device")
        if counts is not None:
            if counts.shape != (b,):
                raise ValueError("counts must have shape [batch]")
            if counts.device != device:
                raise RuntimeError("counts must be on the cache's CUDA device")
            counts = _i64(counts)
        if latent.stride(-1) != 1:
            latent = latent.contiguous()
        if rope.stride(-1) != 1:
            rope = rope.contiguous()
        table, lengths = _i64(self.block_table), _i64(self.lengths)
        with device_guard(device):
            new_lengths = torch.empty(b, dtype=torch.int64, device=device)
            held = torch.empty((b, t, dc), dtype=latent.dtype, device=device) if return_held else None
            a = _lib.FsLatentAppendArgs()
            a.latent, a.rope = latent.data_ptr(), rope.data_ptr()
            a.latent_stride_b, a.latent_stride_t = latent.stride(0), latent.stride(1)
            a.rope_stride_b, a.rope_stride_t = rope.stride(0), rope.stride(1)
            a.dtype = _dtype(latent)
            a.batch, a.tokens, a.latent_dim, a.rope_dim = b, t, dc, dr
            a.page_size, a.table_cols, a.num_pages = page, table.shape[1], pages
            a.block_table, a.lengths = table.data_ptr(), lengths.data_ptr()
            a.counts = counts.data_ptr() if counts is not None else None
            a.values, a.scale, a.ropes = self.values.data_ptr(), self.scale.data_ptr(), self.ropes.data_ptr()
            a.held = held.data_ptr() if held is not None else None
            a.new_lengths = new_lengths.data_ptr()
            a.device_status = status_word(device_status, device)
            _lib.check(_lib.load().fs_latent_append(C.byref(a), stream_of(device)), "fs_latent_append")
        longest = min(int(self.max_seq_len) + t, page * table.shape[1])
        cache = LatentKVCache(self.values, self.scale, self.ropes, self.block_table, new_lengths, longest)
        object.__setattr__(cache, "_checked", True)  # this one's tensors and lengths of the same kind
        return (cache, held) if return_held else cache


def _dtype(t: torch.Tensor) -> int:
    return _lib.FS_BF16 if t.dtype == torch.bfloat16 else _lib.FS_F16


def _check_cache(cache: LatentKVCache) -> None:
    """Raises unless the cache's tensors fit together; once per cache, whose fields are frozen."""
    if getattr(cache, "_checked", False):
        return
    v, s, r = cache.values, cache.scale, cache.ropes
    require_cuda(v, "the latent cache")
    if v.ndim != 3 or v.dtype != torch.int8 or r.ndim != 3 or r.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("a latent cache holds int8 values [P, page, dc] and fp16 or bf16 ropes [P, page, dr]")
    if tuple(s.shape) != tuple(v.shape[:2]) or s.dtype != torch.float32 or tuple(r.shape[:2]) != tuple(v.shape[:2]):
        raise ValueError("scale must be fp32 [P, page] and ropes [P, page, dr] beside values [P, page, dc]")
    if int(v.shape[2]) not in LATENT_DIMS or int(r.shape[2]) not in ROPE_DIMS or int(v.shape[1]) not in LATENT_PAGES:
        raise ValueError(f"latent_dim must be one of {LATENT_DIMS}, rope_dim of {ROPE_DIMS}, the page of {LATENT_PAGES}")
    if int(v.shape[0]) <= 0:
        raise ValueError("a latent cache needs at least one page")
    if not (v.is_contiguous() and s.is_contiguous() and r.is_contiguous()):
        raise ValueError("the latent cache's tensors must be contiguous")
    if any(t.device != v.device for t in (s, r, cache.block_table, cache.lengths)):
        raise RuntimeError("the latent cache's tensors must be on one CUDA device")
    if cache.block_table.ndim != 2 or int(cache.block_table.shape[1]) <= 0 or int(cache.block_table.shape[0]) <= 0 \
            or tuple(cache.lengths.shape) != (int(cache.block_table.shape[0]),):
        raise ValueError("block_table must be [batch, columns] and lengths [batch]")
    object.__setattr__(cache, "_checked", True)


def latent_attention_cuda(q_latent: torch.Tensor, q_rope: torch.Tensor, cache: LatentKVCache, *,
                          sm_scale: Optional[float] = None,
                          device_status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Absorbed attention over a latent cache.

    q_latent [B, T, H, dc] (or [B, H, dc] for one token) and q_rope [B, T, H, dr], in the
    cache's dtype, are the queries of the last T positions of each request (their tokens are
    in the cache already): query t sees the first lengths - T + t + 1 tokens, one that sees
    none gives zeros.  Returns sum_j softmax_j(sm_scale (q_latent . c_j + q_rope . r_j)) c_j
    like q_latent.  sm_scale defaults to 1 / sqrt(dc + dr); a model's own is that of its
    expanded heads, 1 / sqrt(nope + rope).  q_latent takes part as 16-bit fixed point of its
    row (max|q| / 65278 off at most): a dim of q that is hundreds of times the others, over
    latents that are as much smaller, is better moved into the latents before they are stored."""
    _check_cache(cache)
    single = q_latent.ndim == 3
    if single and q_rope.ndim == 3:
        q_latent, q_rope = q_latent.unsqueeze(1), q_rope.unsqueeze(1)
    if q_latent.ndim != 4 or q_rope.ndim != 4 or q_latent.shape[:3] != q_rope.shape[:3]:
        raise ValueError("q_latent and q_rope must be [batch, tokens, heads, dim] (or [batch, heads, dim])")
    b, t, h, dc = q_latent.shape
    pages, page, latent_dim = cache.values.shape
    dr = cache.ropes.shape[2]
    if b != cache.block_table.shape[0] or dc != latent_dim or q_rope.shape[3] != dr:
        raise ValueError("q_latent / q_rope batch and dims must match the cache")
    if t <= 0 or h <= 0:
        raise ValueError("q_latent needs at least one token and one head")
    if q_latent.dtype != cache.ropes.dtype or q_rope.dtype != cache.ropes.dtype:
        raise ValueError("q_latent and q_rope must have the cache's dtype")
    device = cache.values.device
    if q_latent.device != device or q_rope.device != device:
        raise RuntimeError("q_latent and q_rope must be on the cache's CUDA device")
    q, qr = _aligned(q_latent), _aligned(q_rope)
    table, lengths = _i64(cache.block_table), _i64(cache.lengths)
    with device_guard(device):
        out = torch.empty_like(q)
        a = _lib.FsLatentArgs()
        a.q, a.q_rope, a.out = q.data_ptr(), qr.data_ptr(), out.data_ptr()
        a.dtype = _dtype(q)
        a.batch, a.tokens, a.heads, a.latent_dim, a.rope_dim = b, t, h, dc, dr
        a.page_size, a.table_cols = page, table.shape[1]
        a.max_seq_len = _seq_cap(int(cache.max_seq_len), page, table.shape[1])
        a.sm_scale = 1.0 / math.sqrt(dc + dr) if sm_scale is None else float(sm_scale)
        a.num_pages = pages
        a.values, a.scale, a.ropes = cache.values.data_ptr(), cache.scale.data_ptr(), cache.ropes.data_ptr()
        a.block_table, a.lengths = table.data_ptr(), lengths.data_ptr()
        a.device_status = status_word(device_status, device)
        lib, need = _lib.load(), C.c_size_t(0)
        _lib.check(lib.fs_latent_workspace_size(C.byref(a), C.byref(need)), "fs_latent_attention")
        ws = torch.empty(need.value, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
        _lib.check(lib.fs_latent_attention(C.byref(a), stream_of(device)), "fs_latent_attention")
    return out.squeeze(1) if single else out


def latent_prefill_attention_cuda(q: torch.Tensor, kv: torch.Tensor, k_rope: torch.Tensor, q_offsets: torch.Tensor,
                                  k_offsets: torch.Tensor, *, sm_scale: Optional[float] = None,
                                  out: Optional[torch.Tensor] = None,
                                  device_status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Expanded latent attention of packed prompts, causal, aligned at the end.

    q [Nq, H, dn + dr]; kv [Nk, H, dn + dv], every head's key part and value expanded from the
    latents; k_rope [Nk, dr], the rotary key that all heads share (fp16 or bf16, one dtype).
    Request b's queries are rows q_offsets[b] : q_offsets[b + 1] of q, its keys and values rows
    k_offsets[b] : k_offsets[b + 1] (int64 [B + 1] on the device, ascending); its query i of nq
    sees keys j <= i + nk - nq, so a chunk of new tokens sees a cached prefix and, in order,
    itself; a query that sees no key gives zeros.  dn and dv 64 or 128, dr 32 or 64 (dr is read
    from k_rope, dn from q).  Returns out [Nq, H, dv]; a given ``out`` keeps the rows that no
    request covers, otherwise those are zeros.  An infinite or undefined value reaches the
    queries that see its key and no others: infinities of one sign give infinity, else NaN.
    sm_scale defaults to 1 / sqrt(dn + dr)."""
    require_cuda(q, "q")
    if q.ndim != 3 or kv.ndim != 3 or k_rope.ndim != 2:
        raise ValueError("q must be [rows, heads, dim], kv [rows, heads, dim] and k_rope [rows, dim]")
    nq, h, dq = q.shape
    nk, dr = k_rope.shape
    dn = dq - dr
    dv = kv.shape[2] - dn
    if kv.shape[0] != nk or kv.shape[1] != h or h <= 0:
        raise ValueError("kv must have k_rope's rows and q's heads")
    if dn not in (64, 128) or dv not in (64, 128) or dr not in ROPE_DIMS:
        raise ValueError("nope and value dims must be 64 or 128, the rope dim 32 or 64")
    if q.dtype not in (torch.float16, torch.bfloat16) or kv.dtype != q.dtype or k_rope.dtype != q.dtype:
        raise ValueError("q, kv and k_rope must be fp16 or bf16, all of one dtype")
    device = q.device
    if kv.device != device or k_rope.device != device or q_offsets.device != device or k_offsets.device != device:
        raise RuntimeError("q, kv, k_rope and the offsets must be on one CUDA device")
    if q_offsets.ndim != 1 or q_offsets.shape != k_offsets.shape or q_offsets.shape[0] < 2:
        raise ValueError("q_offsets and k_offsets must be [batch + 1]")
    if out is not None:
        if tuple(out.shape) != (nq, h, dv) or out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be a contiguous, 16-byte aligned [Nq, H, dv] tensor of q's dtype")
        if out.device != device:
            raise RuntimeError("out must be on q's CUDA device")
        if any(_overlap(out, t) for t in (q, kv, k_rope)):
            raise ValueError("out must not overlap q, kv or k_rope: other tiles still read them")
    qc, kvc, rc = _aligned(q), _aligned(kv), _aligned(k_rope)
    qo, ko = _i64(q_offsets), _i64(k_offsets)
    with device_guard(device):
        a = _lib.FsLatentPrefillArgs()
        if out is None:
            out, a.clear_rest = torch.empty((nq, h, dv), dtype=q.dtype, device=device), 1
        a.q, a.kv, a.k_rope, a.out = qc.data_ptr(), kvc.data_ptr(), rc.data_ptr(), out.data_ptr()
        a.q_offsets, a.k_offsets = qo.data_ptr(), ko.data_ptr()
        a.q_rows, a.k_rows = nq, nk
        a.dtype, a.batch, a.heads = _dtype(q), int(qo.shape[0]) - 1, h
        a.nope_dim, a.rope_dim, a.value_dim = dn, dr, dv
        a.sm_scale = 1.0 / math.sqrt(dq) if sm_scale is None else float(sm_scale)
        a.device_status = status_word(device_status, device)
        _lib.check(_lib.load().fs_latent_prefill(C.byref(a), stream_of(device)), "fs_latent_prefill")
    return out


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, on a 16-byte boundary (a view into a packed tensor may be neither)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges that two tensors span have a byte in common (strides are
    not negative)."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    span = lambda t: (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()  # noqa: E731
    return a.data_ptr() < b.data_ptr() + span(b) and b.data_ptr() < a.data_ptr() + span(a)
