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

import struct
from typing import NamedTuple, Optional

import torch

from ._lib import DT_BF16, DT_F32, check, lib

HEAD_DIMS = (64, 128, 256)
GROUP = 64  # tokens per value group: page sizes are multiples of it
MAX_PAGE = 1024
MAX_BATCH = 8192
_ROW_DTYPES = {torch.bfloat16: DT_BF16, torch.float32: DT_F32}


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


# The calls below sit in the loop of a decode step, next to kernels of a few microseconds: their checks
# are plain comparisons, and messages are put together only when one fails.
_DESC = struct.Struct("@10q4Q9if")  # dsm_kv8_attn_desc
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _tensor(t: torch.Tensor, name: str, dtype: torch.dtype, shape, dev: int = -1) -> int:
    """``t`` is a contiguous CUDA tensor of that dtype and shape (on device ``dev``); its device."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got {t.dtype} "
                         f"{tuple(t.shape)} with strides {t.stride()}")
    at = t.get_device()
    if dev >= 0 and at != dev:
        raise ValueError(f"{name} is on cuda:{at}, the rest on cuda:{dev}")
    return at


def _page_size(page_size: int) -> int:
    if not (isinstance(page_size, int) and 0 < page_size <= MAX_PAGE and page_size % GROUP == 0):
        raise ValueError(f"page_size must be a multiple of {GROUP}, at most {MAX_PAGE}, got {page_size}")
    return page_size


def _table(table: torch.Tensor, batch: int, dev: int):
    """The row stride and columns of a block table."""
    if not (isinstance(table, torch.Tensor) and table.is_cuda and table.get_device() == dev
            and table.dtype is torch.int32 and table.dim() == 2):
        raise ValueError(f"block_table must be an int32 [{batch}, pages] tensor on cuda:{dev}")
    rows, cols = table.shape
    stride, inner = table.stride()
    if rows != batch or cols < 1 or (inner != 1 and cols > 1) or (batch > 1 and stride < cols):
        raise ValueError(f"block_table must be [{batch}, pages] with contiguous rows that do not overlap, got "
                         f"{tuple(table.shape)} with strides {table.stride()}")
    return max(stride, cols), cols


def _lengths(lengths: torch.Tensor):
    if not (isinstance(lengths, torch.Tensor) and lengths.dim() == 1 and lengths.shape[0] <= MAX_BATCH):
        raise ValueError(f"lengths must be int32 [batch], batch at most {MAX_BATCH}")
    return lengths.shape[0], _tensor(lengths, "lengths", torch.int32, lengths.shape)


def _layer(layer: KV8Layer):
    k, v, ks, vs = layer
    if not (isinstance(k, torch.Tensor) and k.dim() == 4):
        raise ValueError("k_codes must be [n_pages, n_kv, page_size, head_dim]")
    n_pages, n_kv, page, hd = k.shape
    _page_size(page)
    if hd not in HEAD_DIMS or n_pages < 1 or n_kv < 1:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS} and the cache not empty, got {tuple(k.shape)}")
    dev = _tensor(k, "k_codes", torch.uint8, k.shape)
    _tensor(v, "v_codes", torch.uint8, (n_pages, n_kv, page // GROUP, hd, GROUP), dev)
    _tensor(ks, "k_scale", torch.float32, (n_pages, n_kv), dev)
    _tensor(vs, "v_scale", torch.float32, (n_pages, n_kv), dev)
    return n_pages, n_kv, page, hd, dev


def _on_device(fn):
    """Runs ``fn(dev, ...)`` with ``dev`` the current device (the library launches there)."""

    def run(dev: int, *args):
        if _current_device() == dev:
            return fn(dev, *args)
        with torch.cuda.device(dev):
            return fn(dev, *args)

    return run


def paged_extend(lengths: torch.Tensor, new_len: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 n_free: torch.Tensor, page_size: int, max_rows: int) -> PagedRows:
    """Every sequence grows by ``new_len[i]`` tokens: pages off the stack ``free_pages[:n_free]`` go
    into ``block_table``, ``lengths`` and ``n_free`` are updated in place. Returns the step's rows;
    ``max_rows`` (known on the host) bounds them, rows behind the last sequence get slot -1. A
    sequence that finds no pages, table or rows keeps its length and sets the device error word; a page
    outside the pool ends the stack."""
    b, dev = _lengths(lengths)
    _tensor(new_len, "new_len", torch.int32, (b,), dev)
    stride, cols = _table(block_table, b, dev)
    _tensor(free_pages, "free_pages", torch.int32, (free_pages.numel(),), dev)
    _tensor(n_free, "n_free", torch.int32, (1,), dev)
    _page_size(page_size)
    if not 0 <= max_rows <= 0x7FFFFFFF:
        raise ValueError(f"max_rows out of range: {max_rows}")
    return _extend(dev, lengths, new_len, block_table, free_pages, n_free, page_size, max_rows, b, stride, cols)


@_on_device
def _extend(dev, lengths, new_len, block_table, free_pages, n_free, page_size, max_rows, b, stride, cols) -> PagedRows:
    at = lengths.device
    cu_rows = torch.empty(b + 1, dtype=torch.int32, device=at)
    slot_map = torch.empty(max_rows, dtype=torch.int64, device=at)
    positions = torch.empty(max_rows, dtype=torch.int32, device=at)
    rc = lib().dsm_paged_extend(lengths.data_ptr(), new_len.data_ptr(), b, page_size, block_table.data_ptr(), stride,
                                cols, free_pages.data_ptr(), n_free.data_ptr(), free_pages.shape[0],
                                cu_rows.data_ptr(), slot_map.data_ptr(), positions.data_ptr(), max_rows,
                                _raw_stream(dev))
    if rc:
        check(rc, "dsm_paged_extend")
    return PagedRows(cu_rows, slot_map, positions)


def paged_trim(lengths: torch.Tensor, keep_len: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               n_free: torch.Tensor, page_size: int) -> None:
    """Every sequence shrinks to ``min(lengths[i], keep_len[i])`` tokens (0 releases it): its surplus
    pages go back on the stack, ``lengths`` and ``n_free`` are updated in place. Where a table entry is
    outside the pool, nothing is changed and the device error word is set."""
    b, dev = _lengths(lengths)
    _tensor(keep_len, "keep_len", torch.int32, (b,), dev)
    stride, cols = _table(block_table, b, dev)
    _tensor(free_pages, "free_pages", torch.int32, (free_pages.numel(),), dev)
    _tensor(n_free, "n_free", torch.int32, (1,), dev)
    _page_size(page_size)
    _trim(dev, lengths, keep_len, block_table, free_pages, n_free, page_size, b, stride, cols)


@_on_device
def _trim(dev, lengths, keep_len, block_table, free_pages, n_free, page_size, b, stride, cols) -> None:
    rc = lib().dsm_paged_trim(lengths.data_ptr(), keep_len.data_ptr(), b, page_size, block_table.data_ptr(), stride,
                              cols, free_pages.data_ptr(), n_free.data_ptr(), free_pages.shape[0], _raw_stream(dev))
    if rc:
        check(rc, "dsm_paged_trim")


def kv8_append(layer: KV8Layer, k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor) -> None:
    """Writes rows ``k``, ``v`` ``[rows, n_kv, head_dim]`` (bf16 or fp32, any row and head strides)
    into the cache slots ``slot_map`` int64 ``[rows]`` (-1: skipped). Rows of one page must be
    neighbours, as :func:`paged_extend` leaves them, each slot given once."""
    n_pages, n_kv, page, hd, dev = _layer(layer)
    dt = _ROW_DTYPES.get(k.dtype)
    if not (dt is not None and k.dim() == 3 and k.shape[1] == n_kv and k.shape[2] == hd and v.shape == k.shape
            and v.dtype is k.dtype and k.get_device() == dev and v.get_device() == dev):
        raise ValueError(f"k and v must be bf16 or fp32 [rows, {n_kv}, {hd}] tensors on cuda:{dev}, got {k.dtype} "
                         f"{tuple(k.shape)} on {k.device} and {v.dtype} {tuple(v.shape)} on {v.device}")
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError(f"rows of k and v must be {hd} contiguous values")
    _tensor(slot_map, "slot_map", torch.int64, (k.shape[0],), dev)
    _append(dev, layer, k, v, slot_map, dt, n_pages, n_kv, page, hd, ks, vs)


@_on_device
def _append(dev, layer, k, v, slot_map, dt, n_pages, n_kv, page, hd, ks, vs) -> None:
    rc = lib().dsm_kv8_append(k.data_ptr(), v.data_ptr(), dt, k.shape[0], n_kv, hd, ks[0], ks[1], vs[0], vs[1],
                              slot_map.data_ptr(), page, n_pages, layer[0].data_ptr(), layer[1].data_ptr(),
                              layer[2].data_ptr(), layer[3].data_ptr(), _raw_stream(dev))
    if rc:
        check(rc, "dsm_kv8_append")


def gqa_attention_kv8(q: torch.Tensor, layer: KV8Layer, block_table: torch.Tensor, lengths: torch.Tensor,
                      blk_k: Optional[torch.Tensor] = None, blk_v: Optional[torch.Tensor] = None, *,
                      scale: Optional[float] = None) -> torch.Tensor:
    """``q [batch, block, n_heads, head_dim]`` (bf16 or fp32) over each sequence's ``lengths[i]``
    cached rows and then, unless ``blk_k`` is None, the block's own rows ``blk_k`` / ``blk_v``
    ``[batch, n_kv, block, head_dim]``, with no mask; ``scale`` defaults to ``head_dim ** -0.5``.
    Returns ``[batch, block, n_heads * head_dim]`` in q's dtype; a sequence without any row gives
    zeros, and what is not finite in q or the block's rows counts as NaN. q and the block's rows may
    have any strides with contiguous rows."""
    n_pages, n_kv, page, hd, dev = _layer(layer)
    dt = _ROW_DTYPES.get(q.dtype)
    if not (dt is not None and q.dim() == 4 and q.shape[3] == hd and q.get_device() == dev):
        raise ValueError(f"q must be a bf16 or fp32 [batch, block, heads, {hd}] tensor on cuda:{dev}, got {q.dtype} "
                         f"{tuple(q.shape)} on {q.device}")
    b, s, nh, _ = q.shape
    if s < 1 or nh < 1 or nh % n_kv or b > MAX_BATCH:
        raise ValueError(f"q must be [batch <= {MAX_BATCH}, block, a multiple of {n_kv} heads, {hd}], got "
                         f"{tuple(q.shape)}")
    qs = q.stride()
    if (blk_k is None) != (blk_v is None):
        raise ValueError("blk_k and blk_v must both be given or both be None")
    ks = vs = (0, 0, 0, 1)
    if blk_k is not None:
        want = (b, n_kv, s, hd)
        if not (blk_k.shape == want and blk_v.shape == want and blk_k.dtype is q.dtype and blk_v.dtype is q.dtype
                and blk_k.get_device() == dev and blk_v.get_device() == dev):
            raise ValueError(f"blk_k and blk_v must be {q.dtype} {want} tensors on cuda:{dev}, got {blk_k.dtype} "
                             f"{tuple(blk_k.shape)} on {blk_k.device} and {blk_v.dtype} {tuple(blk_v.shape)} on "
                             f"{blk_v.device}")
        ks, vs = blk_k.stride(), blk_v.stride()
    if qs[3] != 1 or ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"rows of q, blk_k and blk_v must be {hd} contiguous values")
    _tensor(lengths, "lengths", torch.int32, (b,), dev)
    stride, cols = _table(block_table, b, dev)
    desc = _DESC.pack(*qs[:3], *ks[:3], *vs[:3], stride, layer[0].data_ptr(), layer[1].data_ptr(), layer[2].data_ptr(),
                      layer[3].data_ptr(), dt, b, s, nh, n_kv, hd, page, n_pages, cols,
                      hd ** -0.5 if scale is None else scale)
    return _attend(dev, desc, q, block_table, lengths, blk_k, blk_v, b, s, nh, n_kv, hd)


@_on_device
def _attend(dev, desc, q, block_table, lengths, blk_k, blk_v, b, s, nh, n_kv, hd) -> torch.Tensor:
    L = lib()
    at = q.device
    out = torch.empty(b, s, nh * hd, dtype=q.dtype, device=at)
    if b == 0:
        return out
    ws_bytes = L.dsm_gqa_attn_kv8_workspace_bytes(b, s, nh, n_kv, hd)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=at)
    rc = L.dsm_gqa_attn_kv8(desc, q.data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
                            None if blk_k is None else blk_k.data_ptr(), None if blk_v is None else blk_v.data_ptr(),
                            out.data_ptr(), ws.data_ptr(), ws_bytes, _raw_stream(dev))
    if rc:
        check(rc, "dsm_gqa_attn_kv8")
    return out


class PagedKVCache:
    """The context caches of ``n_layers`` layers for a batch of sequences: one pool of ``n_pages``
    pages per layer, one block table, one set of lengths.

    A step: ``rows = cache.extend(new_len, max_rows)``; each layer writes its rows with
    ``cache.append(layer, k, v, rows)`` and reads with ``cache.attend(layer, q, blk_k, blk_v)``;
    ``cache.trim(keep_len)`` takes rejected tokens back, and releases finished sequences."""

    def __init__(self, n_layers: int, n_pages: int, n_kv: int, head_dim: int, batch: int, max_pages: int, *,
                 page_size: int = 64, device="cuda"):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if min(n_layers, n_pages, n_kv, batch, max_pages) < 1 or batch > MAX_BATCH:
            raise ValueError(f"sizes must be positive and batch at most {MAX_BATCH}")
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
