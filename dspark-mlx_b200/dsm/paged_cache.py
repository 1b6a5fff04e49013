"""The paged 8-bit KV cache of the Qwen3 draft attention, and its operators.

The reference keeps one dense cache per layer, grown by ``mx.concatenate``, with one context
length for the whole batch (``dspark_mlx/arch/qwen3.py:122-143``, ``:287-296``). Here sequences of
different lengths share a pool of pages, the rows are held as e4m3 codes with one power-of-two
scale per page and KV head, and everything that depends on the lengths is worked out on the GPU:
no call synchronises, and a captured step replays while the lengths change.

* :class:`PagedKVCache` holds the pool, the block table, the lengths and the free pages of a batch
  for every layer; :meth:`PagedKVCache.extend`, :meth:`~PagedKVCache.trim`,
  :meth:`~PagedKVCache.append` and :meth:`~PagedKVCache.attend` are a step's calls.
  ``Qwen3DSparkAttention.append_paged`` / ``attend_paged`` run a layer over it.
* :func:`paged_extend`, :func:`paged_trim`, :func:`kv8_append` and :func:`gqa_attention_kv8` are the
  same operators on plain tensors (the C entry points of the same names, ``include/dsm.h``).

CPU tensors are rejected. What the host cannot see (a pool without free pages, a page id outside
it) sets the device error word: ``dsm._lib.raise_device_error()`` reads it.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from ._lib import KV8AttnDesc, check, dtype_code, lib

HEAD_DIMS = (64, 128, 256)
GROUP = 64  # tokens per value group: page sizes are multiples of it
MAX_PAGE = 1024
MAX_BATCH = 8192


class KV8Layer(NamedTuple):
    """One layer's cache: ``k_codes`` uint8 ``[n_pages, n_kv, page_size, head_dim]`` (from head_dim
    128 on, 16-byte chunk ``c`` of token ``t``'s row at chunk ``c ^ (t & 7)``), ``v_codes`` uint8
    ``[n_pages, n_kv, page_size / 64, head_dim, 64]``, ``k_scale`` / ``v_scale`` fp32
    ``[n_pages, n_kv]``."""

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class PagedRows(NamedTuple):
    """The rows of a step: ``cu_rows`` int32 ``[batch + 1]`` (first row of each sequence),
    ``slot_map`` int64 ``[max_rows]`` (-1: no slot) and ``positions`` int32 ``[max_rows]``."""

    cu_rows: torch.Tensor
    slot_map: torch.Tensor
    positions: torch.Tensor


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _tensor(t: torch.Tensor, name: str, dtype: torch.dtype, shape, device=None) -> None:
    """``shape`` entries that are None are free; the tensor must be contiguous and on the GPU."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    _need(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    _need(t.dim() == len(shape) and all(w is None or w == h for w, h in zip(shape, t.shape)),
          f"{name} must be {['any' if w is None else w for w in shape]}, got {list(t.shape)}")
    _need(t.is_contiguous(), f"{name} must be contiguous")
    _need(device is None or t.device == device, f"{name} is on {t.device}, the rest on {device}")


def _page_size(page_size: int) -> int:
    _need(isinstance(page_size, int) and 0 < page_size <= MAX_PAGE and page_size % GROUP == 0,
          f"page_size must be a multiple of {GROUP}, at most {MAX_PAGE}, got {page_size}")
    return page_size


def _table(block_table: torch.Tensor, batch: int, device) -> None:
    _need(isinstance(block_table, torch.Tensor) and block_table.is_cuda and block_table.device == device,
          f"block_table must be a CUDA tensor on {device}")
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch
          and block_table.shape[1] > 0, f"block_table must be int32 [{batch}, pages]")
    _need(block_table.stride(1) == 1 and (batch < 2 or block_table.stride(0) >= block_table.shape[1]),
          "block_table rows must be contiguous and must not overlap")


def _table_stride(block_table: torch.Tensor) -> int:
    return max(block_table.stride(0), block_table.shape[1])


def _layer(layer: KV8Layer):
    k, v, ks, vs = layer
    _need(isinstance(k, torch.Tensor) and k.dim() == 4, "k_codes must be [n_pages, n_kv, page_size, head_dim]")
    n_pages, n_kv, page, hd = k.shape
    _page_size(page)
    _need(hd in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {hd}")
    _need(n_pages > 0 and n_kv > 0, "an empty cache")
    _tensor(k, "k_codes", torch.uint8, (n_pages, n_kv, page, hd))
    _tensor(v, "v_codes", torch.uint8, (n_pages, n_kv, page // GROUP, hd, GROUP), k.device)
    _tensor(ks, "k_scale", torch.float32, (n_pages, n_kv), k.device)
    _tensor(vs, "v_scale", torch.float32, (n_pages, n_kv), k.device)
    return n_pages, n_kv, page, hd


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def paged_extend(lengths: torch.Tensor, new_len: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 n_free: torch.Tensor, page_size: int, max_rows: int) -> PagedRows:
    """Every sequence grows by ``new_len[i]`` tokens: pages off the stack ``free_pages[:n_free]`` go
    into ``block_table``, ``lengths`` and ``n_free`` are updated in place. Returns the step's rows;
    ``max_rows`` (known on the host) bounds them, rows behind the last sequence get slot -1. A
    sequence that finds no pages, table or rows keeps its length and sets the device error word."""
    _need(isinstance(lengths, torch.Tensor) and lengths.dim() == 1, "lengths must be int32 [batch]")
    b = lengths.shape[0]
    _need(b <= MAX_BATCH, f"batch must be at most {MAX_BATCH}, got {b}")
    _tensor(lengths, "lengths", torch.int32, (b,))
    dev = lengths.device
    _tensor(new_len, "new_len", torch.int32, (b,), dev)
    _table(block_table, b, dev)
    _tensor(free_pages, "free_pages", torch.int32, (None,), dev)
    _tensor(n_free, "n_free", torch.int32, (1,), dev)
    _page_size(page_size)
    _need(0 <= max_rows <= 0x7FFFFFFF, f"max_rows out of range: {max_rows}")
    with torch.cuda.device(dev):
        rows = PagedRows(torch.empty(b + 1, dtype=torch.int32, device=dev),
                         torch.empty(max_rows, dtype=torch.int64, device=dev),
                         torch.empty(max_rows, dtype=torch.int32, device=dev))
        check(lib().dsm_paged_extend(lengths.data_ptr(), new_len.data_ptr(), b, page_size, block_table.data_ptr(),
                                     _table_stride(block_table), block_table.shape[1], free_pages.data_ptr(),
                                     n_free.data_ptr(), free_pages.shape[0], rows.cu_rows.data_ptr(),
                                     rows.slot_map.data_ptr(), rows.positions.data_ptr(), max_rows, _stream(dev)),
              "dsm_paged_extend")
    return rows


def paged_trim(lengths: torch.Tensor, keep_len: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               n_free: torch.Tensor, page_size: int) -> None:
    """Every sequence shrinks to ``min(lengths[i], keep_len[i])`` tokens (0 releases it): its surplus
    pages go back on the stack, ``lengths`` and ``n_free`` are updated in place."""
    _need(isinstance(lengths, torch.Tensor) and lengths.dim() == 1, "lengths must be int32 [batch]")
    b = lengths.shape[0]
    _need(b <= MAX_BATCH, f"batch must be at most {MAX_BATCH}, got {b}")
    _tensor(lengths, "lengths", torch.int32, (b,))
    dev = lengths.device
    _tensor(keep_len, "keep_len", torch.int32, (b,), dev)
    _table(block_table, b, dev)
    _tensor(free_pages, "free_pages", torch.int32, (None,), dev)
    _tensor(n_free, "n_free", torch.int32, (1,), dev)
    _page_size(page_size)
    with torch.cuda.device(dev):
        check(lib().dsm_paged_trim(lengths.data_ptr(), keep_len.data_ptr(), b, page_size, block_table.data_ptr(),
                                   _table_stride(block_table), block_table.shape[1], free_pages.data_ptr(),
                                   n_free.data_ptr(), free_pages.shape[0], _stream(dev)), "dsm_paged_trim")


def kv8_append(layer: KV8Layer, k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor) -> None:
    """Writes rows ``k``, ``v`` ``[rows, n_kv, head_dim]`` (bf16 or fp32, any row and head strides)
    into the cache slots ``slot_map`` int64 ``[rows]`` (-1: skipped). Rows of one page must be
    neighbours, as :func:`paged_extend` leaves them, each slot given once."""
    n_pages, n_kv, page, hd = _layer(layer)
    dev = layer.k_codes.device
    _need(isinstance(k, torch.Tensor) and k.dim() == 3 and tuple(k.shape[1:]) == (n_kv, hd),
          f"k must be [rows, {n_kv}, {hd}]")
    _need(k.dtype in (torch.bfloat16, torch.float32), f"k dtype {k.dtype} unsupported (bf16 or fp32)")
    _need(isinstance(v, torch.Tensor) and v.shape == k.shape and v.dtype == k.dtype,
          "v must have the shape and dtype of k")
    _need(k.device == dev and v.device == dev, f"k and v must be on {dev}")
    _need(k.stride(2) == 1 and v.stride(2) == 1, f"rows of k and v must be {hd} contiguous values")
    _tensor(slot_map, "slot_map", torch.int64, (k.shape[0],), dev)
    with torch.cuda.device(dev):
        check(lib().dsm_kv8_append(k.data_ptr(), v.data_ptr(), dtype_code(k.dtype), k.shape[0], n_kv, hd, k.stride(0),
                                   k.stride(1), v.stride(0), v.stride(1), slot_map.data_ptr(), page, n_pages,
                                   layer.k_codes.data_ptr(), layer.v_codes.data_ptr(), layer.k_scale.data_ptr(),
                                   layer.v_scale.data_ptr(), _stream(dev)), "dsm_kv8_append")


def gqa_attention_kv8(q: torch.Tensor, layer: KV8Layer, block_table: torch.Tensor, lengths: torch.Tensor,
                      blk_k: Optional[torch.Tensor] = None, blk_v: Optional[torch.Tensor] = None, *,
                      scale: Optional[float] = None) -> torch.Tensor:
    """``q [batch, block, n_heads, head_dim]`` (bf16 or fp32) over each sequence's ``lengths[i]``
    cached rows and then, unless ``blk_k`` is None, the block's own rows ``blk_k`` / ``blk_v``
    ``[batch, n_kv, block, head_dim]``, with no mask; ``scale`` defaults to ``head_dim ** -0.5``.
    Returns ``[batch, block, n_heads * head_dim]`` in q's dtype; a sequence without any row gives
    zeros. Every tensor but the cache may have any strides with contiguous rows."""
    n_pages, n_kv, page, hd = _layer(layer)
    dev = layer.k_codes.device
    _need(isinstance(q, torch.Tensor) and q.dim() == 4 and q.shape[3] == hd and q.shape[1] > 0
          and q.shape[2] > 0 and q.shape[2] % n_kv == 0,
          f"q must be [batch, block, a multiple of {n_kv} heads, {hd}]")
    _need(q.dtype in (torch.bfloat16, torch.float32), f"q dtype {q.dtype} unsupported (bf16 or fp32)")
    _need(q.device == dev, f"q must be on {dev}")
    _need(q.stride(3) == 1, f"rows of q must be {hd} contiguous values")
    b, s, nh, _ = q.shape
    _need(b <= MAX_BATCH, f"batch must be at most {MAX_BATCH}, got {b}")
    _need((blk_k is None) == (blk_v is None), "blk_k and blk_v must both be given or both be None")
    for name, t in (("blk_k", blk_k), ("blk_v", blk_v)):
        if t is not None:
            _need(isinstance(t, torch.Tensor) and tuple(t.shape) == (b, n_kv, s, hd) and t.dtype == q.dtype
                  and t.device == dev, f"{name} must be a {q.dtype} [{b}, {n_kv}, {s}, {hd}] tensor on {dev}")
            _need(t.stride(3) == 1, f"rows of {name} must be {hd} contiguous values")
    _tensor(lengths, "lengths", torch.int32, (b,), dev)
    _table(block_table, b, dev)
    L = lib()
    with torch.cuda.device(dev):
        out = torch.empty(b, s, nh * hd, dtype=q.dtype, device=dev)
        if b == 0:
            return out
        ws_bytes = L.dsm_gqa_attn_kv8_workspace_bytes(b, s, nh, n_kv, hd)
        ws = torch.empty(max(1, ws_bytes), dtype=torch.uint8, device=dev)
        bk = (blk_k.stride(0), blk_k.stride(1), blk_k.stride(2)) if blk_k is not None else (0, 0, 0)
        bv = (blk_v.stride(0), blk_v.stride(1), blk_v.stride(2)) if blk_v is not None else (0, 0, 0)
        d = KV8AttnDesc(q.stride(0), q.stride(1), q.stride(2), *bk, *bv, _table_stride(block_table),
                        layer.k_codes.data_ptr(), layer.v_codes.data_ptr(), layer.k_scale.data_ptr(),
                        layer.v_scale.data_ptr(), dtype_code(q.dtype), b, s, nh, n_kv, hd, page, n_pages,
                        block_table.shape[1], float(hd ** -0.5 if scale is None else scale))
        check(L.dsm_gqa_attn_kv8(ctypes.byref(d), q.data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
                                 None if blk_k is None else blk_k.data_ptr(),
                                 None if blk_v is None else blk_v.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes,
                                 _stream(dev)), "dsm_gqa_attn_kv8")
    return out


class PagedKVCache:
    """The context caches of ``n_layers`` layers for a batch of sequences: one pool of ``n_pages``
    pages per layer, one block table, one set of lengths.

    A step: ``rows = cache.extend(new_len, max_rows)``; each layer writes its rows with
    ``cache.append(layer, k, v, rows)`` and reads with ``cache.attend(layer, q, blk_k, blk_v)``;
    ``cache.trim(keep_len)`` takes rejected tokens back, and releases finished sequences."""

    def __init__(self, n_layers: int, n_pages: int, n_kv: int, head_dim: int, batch: int, max_pages: int, *,
                 page_size: int = 64, device="cuda"):
        _need(head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        _need(min(n_layers, n_pages, n_kv, batch, max_pages) > 0, "sizes must be positive")
        _need(batch <= MAX_BATCH, f"batch must be at most {MAX_BATCH}, got {batch}")
        self.page_size = _page_size(page_size)
        self.n_kv, self.head_dim, self.n_pages = n_kv, head_dim, n_pages
        u8 = dict(dtype=torch.uint8, device=device)
        self.k_codes = torch.empty(n_layers, n_pages, n_kv, page_size, head_dim, **u8)
        self.v_codes = torch.empty(n_layers, n_pages, n_kv, page_size // GROUP, head_dim, GROUP, **u8)
        self.k_scale = torch.zeros(n_layers, n_pages, n_kv, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)
        self.block_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=device)

    def layer(self, i: int) -> KV8Layer:
        return KV8Layer(self.k_codes[i], self.v_codes[i], self.k_scale[i], self.v_scale[i])

    def extend(self, new_len: torch.Tensor, max_rows: int) -> PagedRows:
        return paged_extend(self.lengths, new_len, self.block_table, self.free_pages, self.n_free, self.page_size,
                            max_rows)

    def trim(self, keep_len: torch.Tensor) -> None:
        paged_trim(self.lengths, keep_len, self.block_table, self.free_pages, self.n_free, self.page_size)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: PagedRows) -> None:
        kv8_append(self.layer(layer), k, v, rows.slot_map)

    def attend(self, layer: int, q: torch.Tensor, blk_k: Optional[torch.Tensor] = None,
               blk_v: Optional[torch.Tensor] = None, *, scale: Optional[float] = None) -> torch.Tensor:
        return gqa_attention_kv8(q, self.layer(layer), self.block_table, self.lengths, blk_k, blk_v, scale=scale)
