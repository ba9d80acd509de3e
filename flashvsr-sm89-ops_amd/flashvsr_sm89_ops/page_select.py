"""Attention over chosen pages of the 8-bit paged cache (paged_kv.py), on gfx950.

No counterpart in the reference; its draft mask (flashvsr_sm89_ops/lcsa/reference.py:37-64)
scores blocks by pooled bf16 keys, for blocks of queries.  Here each row chooses for itself, by mean
keys that are made once, when a page is full:

    means = page_means(pages)                    # beside the pool, as long as it lives
    # a step:
    q = append_kv(pages, k, v, table, lengths, q=q, ...)
    pool_pages(means, pages, table, lengths, tokens=k.shape[0])
    columns = select_pages(q, means, table, lengths, top=32)
    out = selected_attention(q, pages, table, lengths, columns)

Rows, lengths, tables and cu_tokens are those of append_kv and paged_attention, and like
there nothing is read back: a step captures into a graph.  Inference only: no gradients.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from .paged_kv import (KVPages, _aligned, _cache_arg, _Cache, _check, _check_cache, _check_rows,
                       _check_steps, _one_device)


class PageMeans(NamedTuple):
    """The mean key of every page of a pool (value = mean * scale)."""
    mean: torch.Tensor   # [pages, heads, head_dim] int8
    scale: torch.Tensor  # [pages, heads] float8_e8m0fnu


def page_means(pages: KVPages) -> PageMeans:
    """Means for a pool, all zero: head_dim + 1 bytes a page and head."""
    k = pages.k
    mean = torch.zeros((k.shape[0], k.shape[1], k.shape[3]), dtype=torch.int8, device=k.device)
    scale = torch.zeros(k.shape[:2], dtype=torch.uint8, device=k.device)
    return PageMeans(mean, scale.view(torch.float8_e8m0fnu))


def _check_means(name: str, means: PageMeans):
    mean, scale = means
    _lib.require_dtype(mean, torch.int8, "means.mean")
    _lib.require_dtype(scale, torch.float8_e8m0fnu, "means.scale")
    _check(mean.dim() == 3 and mean.shape[1] > 0 and mean.shape[2] in (64, 128),
           f"{name}: means.mean must be [pages, heads, 64 or 128], got {tuple(mean.shape)}")
    _check(scale.shape == mean.shape[:2],
           f"{name}: means.scale must be {tuple(mean.shape[:2])}, got {tuple(scale.shape)}")
    _check(mean.is_contiguous() and scale.is_contiguous() and mean.data_ptr() % 16 == 0,
           f"{name}: the means must be contiguous, 16-byte aligned")


def pool_pages(means: PageMeans, pages: KVPages, page_table: torch.Tensor, lengths: torch.Tensor,
               cu_tokens: torch.Tensor | None = None, *, tokens: int | None = None) -> PageMeans:
    """Write the mean keys of the pages that have filled up, and return means.

    tokens: the rows of the step (append_kv's k.shape[0]; the n rows of a sequence as
    there): pages that held fewer than 128 tokens before it and hold 128 now.  None: every full
    page of the sequences (cu_tokens does not count then).

    Per page and head scale is the least power of two, 2^-127 or more, of which every |mean|
    is at most 127 times (2^127 for means past that, which are held at 127 of it), and mean the
    nearest integers, ties to even: exactly.  A NaN among a
    head's codes, or as its scale, gives scale NaN.  Page ids outside the pool are passed
    over."""
    r = (_lib._selected_host or _lib.selected_host()).pool_pages(
        means, pages, page_table, lengths, cu_tokens, tokens)
    if r is not None:
        return r
    name = "pool_pages"
    _check(tokens is None or int(tokens) >= 0, f"{name}: tokens {tokens}")
    T = -1 if tokens is None else int(tokens)
    H, D = _check_cache(name, pages, page_table, lengths, cu_tokens, max(T, 0))
    _check_means(name, means)
    N = pages.k.shape[0]
    _check(tuple(means.mean.shape) == (N, H, D),
           f"{name}: means.mean must be {(N, H, D)}, got {tuple(means.mean.shape)}")
    _one_device(name, *pages, *means, page_table, lengths, cu_tokens)
    with torch.cuda.device(page_table.device):
        _lib.check(_lib.lib().fvsr_pool_pages(
            ctypes.byref(_cache_arg(pages, page_table, lengths, cu_tokens)),
            means.mean.data_ptr(), means.scale.data_ptr(), T, _lib.stream(page_table)), name)
    return means


def select_pages(q: torch.Tensor, means: PageMeans, page_table: torch.Tensor,
                 lengths: torch.Tensor, cu_tokens: torch.Tensor | None = None, *, top: int,
                 first: int = 1, recent: int = 1) -> torch.Tensor:
    """The columns of the page table that each row reads: int32 [T, heads, top], rising, -1
    behind the last.

    q [T, q_heads, head_dim] bf16 or fp16, rows as in paged_attention (causal).  A row at
    position p sees the columns 0 .. p // 128.  If they are more than `top`: the first `first` of
    them, the last `recent` (at least 1: that of its own position) and, of those between, the
    top - first - recent whose mean key has the largest product with one of the head's queries.

    The queries of a row and key/value head are rounded to integers of at most 127 times one
    power of two for it; products and scores are then exact, whatever else is in the call, and ties
    go to the lower column.  A page whose mean is NaN, or whose id is outside the pool, comes
    behind all others; for a group of queries with an infinity or NaN all other pages tie.  Rows
    of no sequence get -1.  Tables of up to 32768 columns; of a table far wider than the lengths can
    be, page_table[:, :n] is faster."""
    r = (_lib._selected_host or _lib.selected_host()).select_pages(
        q, means, page_table, lengths, cu_tokens, top, first, recent)
    if r is not None:
        return r
    name = "select_pages"
    _check(q.dim() == 3, f"{name}: q must be [T, heads, head_dim], got {tuple(q.shape)}")
    T, Hq = q.shape[:2]
    _check_means(name, means)
    N, H, D = means.mean.shape
    _check_steps(name, page_table, lengths, cu_tokens, T)
    _check_rows(name, q, None, D, "q")
    _check(Hq > 0 and Hq % H == 0, f"{name}: {Hq} query heads over {H} key/value heads")
    dt = _lib.dtype_code(q, "q")
    if dt == _lib.DT_F32:
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    top, first, recent = int(top), int(first), int(recent)
    _check(first >= 0 and recent >= 1 and first + recent <= top < 1 << 24,
           f"{name}: top {top}, first {first}, recent {recent} (recent at least 1, top at least "
           "first + recent and below 2^24)")
    B, P = page_table.shape
    _check(P <= 32768, f"{name}: {P} table columns, 32768 at most")
    _one_device(name, q, *means, page_table, lengths, cu_tokens)
    with torch.cuda.device(q.device):
        q = _aligned(q)
        out = torch.empty((T, H, top), dtype=torch.int32, device=q.device)
        if B == 0:
            return out.fill_(-1)
        cache = _Cache(None, None, None, None, N, H, D, page_table.data_ptr(),
                       page_table.stride(0) if B > 1 else P, P, lengths.data_ptr(),
                       _lib.ptr(cu_tokens), B)
        _lib.check(_lib.lib().fvsr_select_pages(
            ctypes.byref(cache), means.mean.data_ptr(), means.scale.data_ptr(), q.data_ptr(),
            q.stride(0), q.stride(1), Hq, dt, T, top, first, recent, out.data_ptr(),
            _lib.stream(q)), name)
    return out


def selected_attention(q: torch.Tensor, pages: KVPages, page_table: torch.Tensor,
                       lengths: torch.Tensor, columns: torch.Tensor,
                       cu_tokens: torch.Tensor | None = None, *, sm_scale: float | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * sm_scale) v of each row over the tokens up to its own position in the
    pages that columns names.

    columns int32 [T, heads, n], contiguous: columns of the page table for each row and
    key/value head, in any order.  Entries outside 0 .. p // 128 (p the row's position) are
    passed over; a column that stands twice counts twice.  Everything else as in paged_attention
    with causal=True, precision too: a row that sees nothing is zero, a page id outside the pool
    makes the rows that read it NaN.  There is no gradient: the result asks for none, whatever q does."""
    if out is None:
        r = (_lib._selected_host or _lib.selected_host()).selected_attention(
            q, pages, page_table, lengths, columns, cu_tokens, sm_scale)
        if r is not None:
            return r
    name = "selected_attention"
    _check(q.dim() == 3, f"{name}: q must be [T, heads, head_dim], got {tuple(q.shape)}")
    T, Hq = q.shape[:2]
    H, D = _check_cache(name, pages, page_table, lengths, cu_tokens, T)
    _check_rows(name, q, None, D, "q")
    _check(Hq > 0 and Hq % H == 0, f"{name}: {Hq} query heads over {H} key/value heads")
    dt = _lib.dtype_code(q, "q")
    if dt == _lib.DT_F32:
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    _lib.require_dtype(columns, torch.int32, "columns")
    _check(columns.dim() == 3 and tuple(columns.shape[:2]) == (T, H) and columns.is_contiguous(),
           f"{name}: columns must be a contiguous [{T}, {H}, n], got {tuple(columns.shape)}")
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    _check(0.0 < scale < 3e38, f"{name}: sm_scale must be positive, got {scale}")
    fresh = out is None
    if not fresh:
        _lib.require_dtype(out, q.dtype, "out")
        _check(out.shape == q.shape and out.stride(2) == 1 and out.stride(0) % 4 == 0 and
               out.stride(1) % 4 == 0 and out.data_ptr() % 8 == 0 and
               all(n == 1 or s > 0 for n, s in zip(out.shape, out.stride())),
               f"{name}: out must be {tuple(q.shape)} with 8-byte aligned rows of their own")
    _one_device(name, q, *pages, page_table, lengths, cu_tokens, columns, out)
    with torch.cuda.device(q.device):
        q = _aligned(q)
        if fresh:
            out = (torch.empty if page_table.shape[0] else torch.zeros)(
                q.shape, dtype=q.dtype, device=q.device)
        L, top = _lib.lib(), columns.shape[2]
        cache = ctypes.byref(_cache_arg(pages, page_table, lengths, cu_tokens))
        n = L.fvsr_selected_attn_workspace_floats(cache, T, Hq, top)
        ws = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
        _lib.check(L.fvsr_selected_attn(
            cache, q.data_ptr(), q.stride(0), q.stride(1), Hq, out.data_ptr(), out.stride(0),
            out.stride(1), dt, T, columns.data_ptr(), top, scale, int(fresh), _lib.ptr(ws), n,
            _lib.stream(q)), name)
    return out
