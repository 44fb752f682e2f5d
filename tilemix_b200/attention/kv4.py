"""Paged key/value cache in 4 bits and the attention over it (no counterpart in the reference,
whose sequences under 16 tokens run the model's own attention on a 16-bit cache).

  build_block_tables  pages, slots and positions of the next tokens, from lengths on the device
  release_pages       finished requests' pages go back to the ring of free pages
  kv4_pool            an empty pool: uint8 [pages, kv_heads, page bytes]
  kv4_append          quantise fp16 keys and values and store them at their slots
  kv4_read            read slots back as fp16
  kv4_attention       attention of a few query tokens a request over its cached keys

A value costs 5 bits: 4-bit codes with an fp16 scale and an fp16 minimum for each 32 channels of a
token's head (``value = scale * code + minimum``, ``scale = (max - min) / 15`` rounded down). A slot is
``page * page_size + position in the page``; a request's pages are the entries of its row of the
block table, in order. Every call is asynchronous on the current stream of its tensors' device and
reads nothing back, so a decode step can be captured into a CUDA graph; what only the device can
see (free pages running out, a page number or a slot outside the pool) ends in the device error
word (``tilemix_b200.attention.tilemix.device_error_code``: 11, 12, 13), never in a stray access. The
first call on a device allocates that word and comes before any capture. For inference: no gradient
passes through.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from tilemix_b200._lib import TmBlockTablesParams, TmKv4AttnParams, check, launcher, lib, packer

__all__ = ["BlockTables", "build_block_tables", "release_pages", "kv4_pool", "kv4_append", "kv4_read",
           "kv4_attention"]

_HEAD_DIMS = (64, 128)
_MAX_KEYS = 2**30  # of a request
_MAX_SCALE = 2.0 ** 80  # every score of fp16 rows stays finite in fp32
_pack_tables = packer(TmBlockTablesParams)
_pack_attn = packer(TmKv4AttnParams)
_launch_tables, _launch_release = launcher("tm_build_block_tables"), launcher("tm_release_pages")
_launch_append, _launch_read = launcher("tm_kv4_append"), launcher("tm_kv4_read")
_launch_attn = launcher("tm_kv4_attn")


class BlockTables(NamedTuple):
    """What :func:`build_block_tables` returns (device tensors)."""

    slots: Tensor          # int64 [max_new_tokens]: slot of each new token, -1 behind the last one
    positions: Tensor      # int32 [max_new_tokens]: its position in its request (0 behind the last one)
    cu_seqlens_q: Tensor   # int32 [batch + 1]: row offsets of the requests' new tokens
    kv_lens: Tensor        # int32 [batch]: tokens in the cache once the new ones are stored
    free_span: Tensor      # int64 [2]: the ring's free entries after this call


def _check_page_size(page_size: int) -> None:
    if page_size < 16 or page_size % 16:
        raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")


def _check(name: str, t: Tensor, dtype: torch.dtype, index: int, ndim: int = 1) -> None:
    """A control tensor of a call on CUDA device ``index``: its type, device and layout."""
    if t.dtype is dtype and t.ndim == ndim and t.get_device() == index and (t.stride(-1) == 1 or not t.numel()):
        return
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}")
    if t.get_device() != index:
        raise ValueError("all tensors of a call must share one CUDA device")
    raise ValueError(f"{name} must have {ndim} dimension{'s' * (ndim > 1)}, the last one contiguous")


def build_block_tables(cached_lens: Tensor, new_lens: Tensor, block_table: Tensor, free_pages: Tensor,
                       free_span: Tensor, *, page_size: int, max_new_tokens: int) -> BlockTables:
    """Pages and slots for the next tokens of a batch, from lengths that live on the device.

    ``cached_lens`` / ``new_lens`` int32 [batch]: tokens in the cache and tokens to add (0 allowed).
    ``block_table`` int32 [batch, columns]: a request's pages so far; its new pages are entered in
    place. ``free_pages`` int32 [capacity]: a ring of free page numbers, of which the entries
    ``[free_span[0], free_span[1])`` (int64 [2], modulo the capacity) are free; pages are taken from
    the front, in request order. ``max_new_tokens``: rows of the packed new tokens (their sum, or
    more: the rows behind the last request get slot -1, which :func:`kv4_append` skips).

    ``cached_lens`` and ``free_span`` are not changed: the caller carries ``kv_lens`` and the returned
    ``free_span`` on to the next step. If the free pages, the table's columns or ``max_new_tokens``
    do not suffice, or a length is negative, nothing is allocated (every slot -1, ``kv_lens`` the
    cached lengths, offsets 0, ``free_span`` unchanged) and ``device_error_code`` reports 11.
    """
    if not cached_lens.is_cuda:
        raise RuntimeError("the block tables are built by a CUDA kernel")
    index = cached_lens.get_device()
    _check("cached_lens", cached_lens, torch.int32, index)
    _check("new_lens", new_lens, torch.int32, index)
    _check("block_table", block_table, torch.int32, index, 2)
    _check("free_pages", free_pages, torch.int32, index)
    _check("free_span", free_span, torch.int64, index)
    _check_page_size(page_size)
    batch = cached_lens.numel()
    if new_lens.numel() != batch or block_table.shape[0] != batch or free_span.numel() != 2:
        raise ValueError("cached_lens, new_lens and block_table must agree on the batch, free_span has two entries")
    if batch > 8192:
        raise ValueError("at most 8192 requests")
    if not 0 <= max_new_tokens < 2**31:
        raise ValueError("max_new_tokens must be in [0, 2^31)")
    # one allocation, slots and positions on 16 bytes
    n, wide = 2 * max_new_tokens, (max_new_tokens + 3) // 4 * 8
    slots, _, span, positions, cu, kv_lens = cached_lens.new_empty(
        wide + 4 + max_new_tokens + 2 * batch + 1).split_with_sizes((n, wide - n, 4, max_new_tokens, batch + 1, batch))
    slots, span = slots.view(torch.int64), span.view(torch.int64)
    _launch_tables(index, _pack_tables(
        cached_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        free_pages.data_ptr(), free_pages.numel(), free_span.data_ptr(), batch, page_size, max_new_tokens,
        slots.data_ptr(), positions.data_ptr(), cu.data_ptr(), kv_lens.data_ptr(), span.data_ptr()))
    return BlockTables(slots, positions, cu, kv_lens, span)


def release_pages(lens: Tensor, done: Tensor, block_table: Tensor, free_pages: Tensor, free_span: Tensor, *,
                  page_size: int) -> None:
    """Give the pages of finished requests back, in place: where ``done`` (bool [batch]) is set, the
    pages of ``lens[b]`` (int32) tokens go to the ring's end in request order, the request's table
    entries become -1 and its length 0; ``free_span[1]`` grows by their number."""
    if not lens.is_cuda:
        raise RuntimeError("the pages are released by a CUDA kernel")
    index = lens.get_device()
    _check("lens", lens, torch.int32, index)
    _check("done", done, torch.bool, index)
    _check("block_table", block_table, torch.int32, index, 2)
    _check("free_pages", free_pages, torch.int32, index)
    _check("free_span", free_span, torch.int64, index)
    _check_page_size(page_size)
    batch = lens.numel()
    if done.numel() != batch or block_table.shape[0] != batch or free_span.numel() != 2:
        raise ValueError("lens, done and block_table must agree on the batch, free_span has two entries")
    _launch_release(index, lens.data_ptr(), done.data_ptr(), block_table.data_ptr(), block_table.stride(0),
                    block_table.shape[1], free_pages.data_ptr(), free_pages.numel(), free_span.data_ptr(), batch, page_size)


def _page_bytes(page_size: int, head_dim: int) -> int:
    return page_size // 16 * 20 * head_dim


def kv4_pool(num_pages: int, page_size: int, kv_heads: int, head_dim: int, device=None) -> Tensor:
    """An empty pool, uint8 ``[num_pages, kv_heads, page bytes]`` (1.25 bytes a channel of K and V)."""
    _check_page_size(page_size)
    if head_dim not in _HEAD_DIMS:
        raise ValueError("the 4-bit cache supports head_dim 64 and 128")
    if num_pages < 0 or kv_heads <= 0:
        raise ValueError("num_pages must not be negative and kv_heads must be positive")
    return torch.zeros((num_pages, kv_heads, _page_bytes(page_size, head_dim)), dtype=torch.uint8,
                       device="cuda" if device is None else device)


def _pool_pages(pool: Tensor, heads: Optional[int], head_dim: int, index: int) -> tuple[int, int, int]:
    """(pages, KV heads, page size) of a pool that holds ``heads`` KV heads of ``head_dim``; raises if it cannot."""
    if head_dim not in _HEAD_DIMS:
        raise ValueError("the 4-bit cache supports head_dim 64 and 128")
    if pool.dtype is not torch.uint8 or pool.ndim != 3 or not pool.is_contiguous():
        raise TypeError("pool must be a contiguous uint8 [pages, kv_heads, page bytes] tensor (kv4_pool)")
    if pool.get_device() != index:
        raise ValueError("all tensors of a call must share one CUDA device")
    pages, heads_k, row = pool.shape
    if heads is not None and heads_k != heads:
        raise ValueError(f"pool has {heads_k} KV heads, expected {heads}")
    if row == 0 or row % (20 * head_dim):
        raise ValueError(f"a pool row of {row} bytes does not hold whole blocks of head_dim {head_dim}")
    return pages, heads_k, row // (20 * head_dim) * 16


def kv4_append(k: Tensor, v: Tensor, pool: Tensor, slots: Tensor) -> None:
    """Quantise fp16 ``k`` / ``v`` [tokens, kv_heads, head_dim] and store token i at ``slots[i]`` (int64;
    -1 is skipped). Rows may be strided; the head dimension is contiguous and rows start on 16
    bytes. The slots of one call are distinct. A group of 32 channels with an infinity or a NaN
    reads back as NaN."""
    if not k.is_cuda:
        raise RuntimeError("the cache is written by a CUDA kernel")
    index = k.get_device()
    if k.ndim != 3 or v.ndim != 3:
        raise ValueError("expected [tokens, kv_heads, head_dim] tensors")
    if v.shape != k.shape:
        raise ValueError("K and V shapes must match")
    if v.get_device() != index:
        raise ValueError("all tensors of a call must share one CUDA device")
    if k.dtype != torch.float16 or v.dtype != torch.float16:
        raise TypeError("the sm_100a cache kernels take fp16; k and v must be torch.float16")
    n, heads, d = k.shape
    pages, _, page_size = _pool_pages(pool, heads, d, index)
    _check("slots", slots, torch.int64, index)
    if slots.numel() != n:
        raise ValueError(f"{slots.numel()} slots for {n} tokens")
    k_tok, k_head, k_dim = k.stride()
    v_tok, v_head, v_dim = v.stride()
    if n and (k_dim != 1 or v_dim != 1):
        raise ValueError("the head dimension must be contiguous")
    _launch_append(index, k.data_ptr(), k_tok, k_head, v.data_ptr(), v_tok, v_head, n, slots.data_ptr(),
                   pool.data_ptr(), pages, heads, d, page_size)


def kv4_read(pool: Tensor, slots: Tensor, head_dim: int) -> tuple[Tensor, Tensor]:
    """The cached keys and values at ``slots`` (int64; -1 gives zeros) as fp16 [slots, kv_heads, head_dim]."""
    if not pool.is_cuda:
        raise RuntimeError("the cache is read by a CUDA kernel")
    index = pool.get_device()
    pages, heads, page_size = _pool_pages(pool, None, head_dim, index)
    _check("slots", slots, torch.int64, index)
    n = slots.numel()
    k, v = pool.new_empty((2, n, heads, 2 * head_dim)).view(torch.float16)
    _launch_read(index, pool.data_ptr(), pages, heads, head_dim, page_size, slots.data_ptr(), n, k.data_ptr(),
                 v.data_ptr())
    return k, v


def kv4_attention(q: Tensor, pool: Tensor, block_table: Tensor, kv_lens: Tensor,
                  cu_seqlens_q: Optional[Tensor] = None, max_seqlen_q: int = 1, *, sm_scale: Optional[float] = None,
                  causal: bool = True, key_mask: Optional[Tensor] = None, max_kv_len: Optional[int] = None,
                  out: Optional[Tensor] = None) -> Tensor:
    """Attention of the new tokens' queries over the cached keys (their own among them).

    ``q`` fp16 [rows, heads, head_dim] packs the requests' query tokens; ``cu_seqlens_q`` int32
    [batch + 1] delimits them and ``max_seqlen_q`` bounds their number (without ``cu_seqlens_q``: one
    row a request). ``kv_lens`` int32 [batch]: cached keys of each request. With ``causal`` the i-th
    of a request's n query tokens sees the keys up to position ``kv_len - n + i``. ``key_mask`` (bool
    [batch, columns], optional) excludes keys for every row of a request; a key behind its last
    column is excluded too. A row that sees no key is 0. ``max_kv_len`` bounds ``kv_lens`` on the
    host (default: the table's capacity, at most 2^30); a small bound makes for a small launch. Keys
    beyond it, or query tokens beyond ``max_seqlen_q``, are left out and move nothing for the others;
    a request whose offsets are not rows of ``q`` in order is left out whole, a negative length
    counts as 0 (``device_error_code`` 11 for all of these). Rows of ``q`` that belong to no request
    are left as they were in ``out`` (without ``out`` they hold anything).
    """
    if not q.is_cuda:
        raise RuntimeError("the cache attention is a CUDA kernel")
    index = q.get_device()
    if q.ndim != 3:
        raise ValueError("expected q [rows, heads, head_dim]")
    if q.dtype is not torch.float16:
        raise TypeError("the sm_100a cache kernels take fp16; q must be torch.float16")
    rows, heads, d = q.shape
    pages, heads_k, page_size = _pool_pages(pool, None, d, index)
    if heads_k == 0 or heads % heads_k:
        raise ValueError("Q heads must be divisible by KV heads")
    _check("block_table", block_table, torch.int32, index, 2)
    _check("kv_lens", kv_lens, torch.int32, index)
    batch, cols = block_table.shape
    if kv_lens.numel() != batch:
        raise ValueError("block_table and kv_lens must agree on the batch")
    if rows and max_seqlen_q < 1:
        raise ValueError("max_seqlen_q must be positive")
    if cu_seqlens_q is not None:
        _check("cu_seqlens_q", cu_seqlens_q, torch.int32, index)
        if cu_seqlens_q.numel() != batch + 1:
            raise ValueError("cu_seqlens_q must have batch + 1 entries")
    elif rows != batch or max_seqlen_q != 1:
        raise ValueError("without cu_seqlens_q there is one query row a request")
    if key_mask is not None:
        _check("key_mask", key_mask, torch.bool, index, 2)
        if key_mask.shape[0] != batch:
            raise ValueError("key_mask must have a row for each request")
    q_tok, q_head, q_dim = q.stride()
    if rows and q_dim != 1:
        raise ValueError("the head dimension must be contiguous")
    if out is None:
        out, o_tok, o_head = q.new_empty((rows, heads, d)), heads * d, d
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.get_device() != index or (rows and out.stride(2) != 1):
            raise ValueError("out must match q")
        o_tok, o_head, _ = out.stride()
    scale = d ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0 < scale <= _MAX_SCALE:
        raise ValueError("sm_scale must be positive and at most 2^80")
    capacity = min(cols * page_size, _MAX_KEYS)
    bound = capacity if max_kv_len is None else min(max(int(max_kv_len), 0), capacity)
    mask = (0, 0, 0) if key_mask is None else (key_mask.data_ptr(), key_mask.stride(0), key_mask.shape[1])
    # From the allocator on the call's own stream: two streams or graphs never share it.
    nbytes = _workspace_bytes(batch, heads, heads_k, d, max_seqlen_q, bound)
    work = pool.new_empty(nbytes)
    _launch_attn(index, _pack_attn(
        q.data_ptr(), q_tok, q_head, out.data_ptr(), o_tok, o_head, rows, pool.data_ptr(), pages,
        block_table.data_ptr(), block_table.stride(0), cols, page_size, kv_lens.data_ptr(),
        0 if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), *mask, batch, heads, heads_k, d, max_seqlen_q, bound,
        bool(causal), scale), work.data_ptr(), nbytes)
    return out


@lru_cache(maxsize=256)
def _workspace_bytes(batch: int, heads: int, heads_k: int, d: int, max_seqlen_q: int, bound: int) -> int:
    """Workspace of an attention call; it depends on these sizes alone (the others and the pointers stand in)."""
    at, need = 1 << 20, ctypes.c_int64()
    args = _pack_attn(at, d, d, at, d, d, max(batch, 1), at, 1, at, 1, 1, 16, at, at, 0, 0, 0, batch, heads, heads_k, d,
                      max_seqlen_q, bound, 1, 1.0)
    check(lib().tm_kv4_attn_workspace(args, ctypes.byref(need)), "tm_kv4_attn")
    return need.value
