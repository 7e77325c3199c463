"""A paged key/value cache: block tables, slot maps and stores.

A cache is a pair of tensors (num_pages, page_size, heads, head_dim), or any
strided view of that shape (heads before slots, layers interleaved); slot s is
row s % page_size of page s // page_size. A request's block table lists its
pages in order. One serving step runs

    m = map_step(cached_lens, new_lens, page_counts, block_tables, free_pages, num_free,
                 page_size=..., num_tokens=...)
    write_kv(k, v, k_cache, v_cache, m.slots)
    attention.attention_tree(q, k_cache, v_cache, block_tables, m.seq_lens, m.cu_seqlens, ...)

without a host read: lengths, tables and the free list stay on the GPU. Every
call is asynchronous on the current stream; what a kernel finds wrong is
reported by ``ops.check_status``.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .ops import _require_cuda, _stream_handle, status_tensor

_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
_I64x10 = ctypes.c_int64 * 10
_ONE = torch.Size([1])


class StepMaps(NamedTuple):
    """Where a step's new tokens go (see map_step)."""

    slots: torch.Tensor        # int64 (num_tokens,)
    positions: torch.Tensor    # int32 (num_tokens,)
    cu_seqlens: torch.Tensor   # int32 (requests + 1,)
    seq_lens: torch.Tensor     # int32 (requests,)
    page_counts: torch.Tensor  # int32 (requests,)
    num_free: torch.Tensor     # int32 (1,)


def _int_vector(t: torch.Tensor, n: int | None, dtype: torch.dtype, name: str) -> torch.Tensor:
    shape = t.shape
    if t.dtype is not dtype or len(shape) != 1 or (n is not None and shape[0] != n):
        want = "" if n is None else f"{n} "
        raise ValueError(f"{name} must be a 1-D tensor of {want}{dtype}, got {tuple(t.shape)} {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def map_step(cached_lens: torch.Tensor, new_lens: torch.Tensor, page_counts: torch.Tensor,
             block_tables: torch.Tensor, free_pages: torch.Tensor, num_free: torch.Tensor, *,
             page_size: int, num_tokens: int) -> StepMaps:
    """Takes the pages that a step needs and maps its new tokens to slots.

    Request r has ``cached_lens[r]`` tokens in the cache, ``page_counts[r]`` pages
    in row r of ``block_tables`` (requests, max_pages) and ``new_lens[r]`` new
    tokens. The pages that it lacks come off the top of the stack
    ``free_pages[:num_free]``, request by request, and are appended to its row in
    place. ``num_tokens`` is the number of packed new tokens (or more: rows past
    the last token get slot -1). Everything else comes back as new tensors, so a
    step can be planned again from the same inputs.

    When the list runs out, the missing table entries and slots are -1 and the
    returned ``num_free`` is minus the number of missing pages. All lengths,
    counts and tables are int32 CUDA tensors, ``num_free`` of shape (1,). At most
    8192 requests."""
    dev = _require_cuda(cached_lens, new_lens, page_counts, block_tables, free_pages, num_free)
    i32 = torch.int32
    if block_tables.dtype is not i32 or len(block_tables.shape) != 2:
        raise ValueError("block_tables must be a 2-D int32 tensor")
    per_request = block_tables.shape[:1]
    requests, max_pages = block_tables.shape
    table_stride, column_stride = block_tables.stride()
    if max_pages > 1 and column_stride != 1:
        raise ValueError("block_tables is updated in place: its rows must be contiguous")
    if not (cached_lens.dtype is new_lens.dtype is page_counts.dtype is free_pages.dtype is num_free.dtype is i32
            and cached_lens.shape == new_lens.shape == page_counts.shape == per_request
            and len(free_pages.shape) == 1 and num_free.shape == _ONE
            and cached_lens.is_contiguous() and new_lens.is_contiguous()
            and page_counts.is_contiguous() and free_pages.is_contiguous()):
        cached_lens = _int_vector(cached_lens, requests, i32, "cached_lens")
        new_lens = _int_vector(new_lens, requests, i32, "new_lens")
        page_counts = _int_vector(page_counts, requests, i32, "page_counts")
        free_pages = _int_vector(free_pages, None, i32, "free_pages")
        num_free = _int_vector(num_free, 1, i32, "num_free")
    if page_size < 1 or num_tokens < 0:
        raise ValueError("page_size must be positive and num_tokens not negative")
    # one allocation for the int32 outputs
    n = num_tokens
    slots = block_tables.new_empty(n, dtype=torch.int64)
    ints = block_tables.new_empty(n + 3 * requests + 2)
    positions, cu, seq, counts, left = ints.unsafe_split_with_sizes(
        (n, requests + 1, requests, requests, 1))
    base = ints.data_ptr()
    rc = _lib.lib().b2g_kv_map_step(
        cached_lens.data_ptr(), new_lens.data_ptr(), page_counts.data_ptr(),
        block_tables.data_ptr(), table_stride, requests, max_pages,
        free_pages.data_ptr(), free_pages.shape[0], num_free.data_ptr(), page_size, n,
        slots.data_ptr(), base, base + 4 * n, base + 4 * (n + requests + 1),
        base + 4 * (n + 2 * requests + 1), base + 4 * (n + 3 * requests + 1),
        status_tensor(dev).data_ptr(), _stream_handle(dev))
    _lib.check(rc, "b2g_kv_map_step")
    return StepMaps(slots, positions, cu, seq, counts, left)


def check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, dtype: torch.dtype) -> None:
    """Both caches 4-D, of one shape and ``dtype``, with unit stride along the head dim."""
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must share one shape (pages, page_size, heads, head_dim)")
    if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError(f"the caches must hold {dtype}, got {k_cache.dtype} and {v_cache.dtype}")
    if shape[3] > 1 and (k_cache.stride(3) != 1 or v_cache.stride(3) != 1):
        raise ValueError("the caches must be contiguous along the head dim")


def write_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             slots: torch.Tensor) -> None:
    """Stores ``k`` and ``v`` (tokens, heads, head_dim) at ``slots`` (int64, one per
    token) of the caches. Negative slots are skipped; a slot past the cache is
    skipped and reported by ``ops.check_status``. ``k`` and ``v`` may be views of a
    fused projection's output (unit stride along the head dim)."""
    dev = _require_cuda(k, v, k_cache, v_cache, slots)
    dtype = _DT.get(k.dtype)
    if dtype is None or v.dtype is not k.dtype:
        raise ValueError("k and v must share one dtype, float16 or bfloat16")
    if len(k.shape) != 3 or k.shape != v.shape:
        raise ValueError("k and v must share one shape (tokens, heads, head_dim)")
    check_caches(k_cache, v_cache, k.dtype)
    tokens, heads, dim = k.shape
    pages, page, cache_heads, cache_dim = k_cache.shape
    if (cache_heads, cache_dim) != (heads, dim):
        raise ValueError(f"k has {heads} heads of {dim}, the cache {cache_heads} of {cache_dim}")
    slots = _int_vector(slots, tokens, torch.int64, "slots")
    if tokens == 0:
        return
    (k_token, k_head, k_dim), (v_token, v_head, v_dim) = k.stride(), v.stride()
    if k_dim != 1 or v_dim != 1:
        k, v = k.contiguous(), v.contiguous()
        k_token = v_token = heads * dim
        k_head = v_head = dim
    strides = _I64x10(k_token, k_head, v_token, v_head, *k_cache.stride()[:3],
                      *v_cache.stride()[:3])
    rc = _lib.lib().b2g_kv_write(
        k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), strides,
        slots.data_ptr(), tokens, heads, dim, pages, page, dtype,
        status_tensor(dev).data_ptr(), _stream_handle(dev))
    _lib.check(rc, "b2g_kv_write")
