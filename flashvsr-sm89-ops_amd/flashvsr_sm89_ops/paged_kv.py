"""An 8-bit key/value cache in pages, and the attention that reads it, on gfx950.

No counterpart in the reference, whose self-attention keeps the windows of the
chunks before in bf16 (flashvsr_sm89_ops/integrate.py:59-83).  A page is 128 tokens, the
attention's key block; per page and key/value head the codes are e4m3 and share
one power-of-two scale (e8m0).  A page table says which pages hold a sequence, so
sequences of any lengths share one pool:

    pages = kv_pages(1000, heads=8, head_dim=128, device="cuda")
    lengths += 1                                 # the new tokens included
    q = append_kv(pages, k, v, table, lengths, freqs_cis=freqs, positions=pos, q=q)
    out = paged_attention(q, pages, table, lengths)

Both take a step of any mix: ``[T, heads, head_dim]`` rows packed by
``cu_tokens`` (int32 [B + 1], from 0 and never falling), or, without it, the same number
for every sequence (one each: the next token).  Lengths, table and cu_tokens stay on the
device and are never read back, so a step can be captured into a graph and replayed as
they change.  How a call's work is cut up follows from its sizes alone, the table's width among
them; a table far wider than the lengths costs some time.  Inference only: no gradients.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib

PAGE = 128
_HEAD_DIMS = (64, 128)


class KVPages(NamedTuple):
    """The pool: codes and scales of every page (value = code * scale).  v lies
    [dim, token], so that both are read as the matrix cores take them."""
    k: torch.Tensor        # [pages, heads, 128, head_dim] float8_e4m3fn
    v: torch.Tensor        # [pages, heads, head_dim, 128] float8_e4m3fn
    k_scale: torch.Tensor  # [pages, heads] float8_e8m0fnu
    v_scale: torch.Tensor  # [pages, heads] float8_e8m0fnu


def kv_pages(pages: int, heads: int, head_dim: int = 128, device="cuda") -> KVPages:
    """A pool of empty pages: 256 * head_dim bytes and two scales a page and head."""
    if pages < 0 or heads <= 0 or head_dim not in _HEAD_DIMS:
        raise ValueError(f"kv_pages: pages {pages}, heads {heads}, head_dim {head_dim} (64 or 128)")

    def zeros(dtype, *shape):
        return torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
    e4m3, e8m0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return KVPages(zeros(e4m3, pages, heads, PAGE, head_dim),
                   zeros(e4m3, pages, heads, head_dim, PAGE),
                   zeros(e8m0, pages, heads), zeros(e8m0, pages, heads))


def _check(ok: bool, what: str):
    if not ok:
        raise ValueError(what)


def _check_steps(name: str, table, lengths, cu, T: int):
    """Page table, lengths and cu_tokens of a call with T rows."""
    for t, n in ((table, "page_table"), (lengths, "lengths"), (cu, "cu_tokens")):
        if t is not None:
            _lib.require_dtype(t, torch.int32, n)
    _check(table.dim() == 2 and (table.shape[1] <= 1 or table.stride(1) == 1) and
           (table.shape[0] <= 1 or table.stride(0) >= table.shape[1]),
           f"{name}: page_table must be [sequences, pages] with unit-stride rows")
    B = table.shape[0]
    _check(tuple(lengths.shape) == (B,) and lengths.is_contiguous(),
           f"{name}: lengths must be a contiguous [{B}]")
    if cu is not None:
        _check(tuple(cu.shape) == (B + 1,) and cu.is_contiguous(),
               f"{name}: cu_tokens must be a contiguous [{B + 1}]")
    else:
        _check(T % B == 0 if B else T == 0,
               f"{name}: {T} rows are not the same number for each of {B} sequences (give "
               "cu_tokens)")


def _check_cache(name: str, pages: KVPages, table, lengths, cu, T: int):
    k, v, ks, vs = pages
    _check(k.dim() == 4 and k.shape[2] == PAGE and k.shape[3] in _HEAD_DIMS and k.shape[1] > 0,
           f"{name}: pages.k must be [pages, heads, {PAGE}, 64 or 128], got {tuple(k.shape)}")
    N, H, _, D = k.shape
    _check(tuple(v.shape) == (N, H, D, PAGE) and tuple(ks.shape) == (N, H) == tuple(vs.shape),
           f"{name}: pages.v must be {(N, H, D, PAGE)} and the scales {(N, H)}, got "
           f"{tuple(v.shape)}, {tuple(ks.shape)}, {tuple(vs.shape)}")
    for t, n in ((k, "pages.k"), (v, "pages.v")):
        _lib.require_dtype(t, torch.float8_e4m3fn, n)
    for t, n in ((ks, "pages.k_scale"), (vs, "pages.v_scale")):
        _lib.require_dtype(t, torch.float8_e8m0fnu, n)
    _check(all(t.is_contiguous() for t in pages), f"{name}: the pages must be contiguous")
    _check_steps(name, table, lengths, cu, T)
    return H, D


def _check_rows(name: str, x: torch.Tensor, heads, D: int, what: str):
    _check(x.dim() == 3 and x.shape[2] == D and (heads is None or x.shape[1] == heads),
           f"{name}: {what} must be [T, {heads or 'heads'}, {D}], got {tuple(x.shape)}")


def _one_device(name: str, *ts):
    ts = [t for t in ts if t is not None]
    _lib.require_gpu(*ts)
    _check(all(t.device == ts[0].device for t in ts), f"{name}: tensors on several devices")


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x with 16-byte aligned rows, copied if it has not: what the kernels load."""
    size = x.element_size()
    ok = x.stride(-1) == 1 or x.shape[-1] == 1
    if ok and x.data_ptr() % 16 == 0 and all(s * size % 16 == 0 for s in x.stride()[:-1]):
        return x
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


class _Cache(ctypes.Structure):
    """fvsr_kv_cache."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] +
                [(n, ctypes.c_int64) for n in ("pages", "heads", "head_dim")] +
                [("table", ctypes.c_void_p)] +
                [(n, ctypes.c_int64) for n in ("table_stride", "table_pages")] +
                [("lengths", ctypes.c_void_p), ("cu", ctypes.c_void_p),
                 ("sequences", ctypes.c_int64)])


def _cache_arg(pages: KVPages, table, lengths, cu):
    k = pages.k
    B, P = table.shape
    return _Cache(k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(),
                  pages.v_scale.data_ptr(), k.shape[0], k.shape[1], k.shape[3], table.data_ptr(),
                  table.stride(0) if B > 1 else P, P, lengths.data_ptr(), _lib.ptr(cu), B)


def _norm(name: str, weight, heads: int, D: int, what: str) -> int:
    if weight is None:
        return _lib.NORM_NONE
    if weight.numel() == D:
        return _lib.NORM_HEAD
    _check(weight.numel() == heads * D,
           f"{name}: {what} has {weight.numel()} elements, a head {D}, a row {heads * D}")
    return _lib.NORM_ROW


def _rotations(freqs: torch.Tensor) -> torch.Tensor:
    """complex [.., rows, D / 2] -> fp32 [rows, D / 2, 2] (cos, sin): a contiguous complex64 table
    itself, any other converted by this call (and so by every replay of a captured one)."""
    f = freqs.reshape(-1, freqs.shape[-1]).resolve_conj()
    return torch.view_as_real(f.to(torch.complex64).contiguous())


def append_kv(pages: KVPages, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, cu_tokens: torch.Tensor | None = None, *, freqs_cis=None,
              positions: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
              q: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
              eps: float = 1e-6):
    """Write the step's keys and values into their pages; the rotated q, if
    given, is returned.

    k, v [T, heads, head_dim] and q [T, q_heads, head_dim], all bf16, fp16 or fp32; rows
    may be strided (columns of a fused qkv).  The n rows of sequence b go to
    positions lengths[b] - n .. lengths[b] - 1 (lengths [B] int32: with this
    step's tokens), position p to slot p % 128 of page page_table[b, p // 128]
    (int32 [B, P]).  Positions below 0 or past the table and pages outside the pool
    are not stored; rows behind cu_tokens[B] belong to nobody (their q is turned all the
    same).

    k_weight, q_weight: RMSNorm first, over each head ([head_dim]) or the whole
    row ([heads * head_dim]).  freqs_cis (complex [rows, head_dim / 2]; complex64 is read as it
    lies, complex128 converted by each call): then the pairs (2i, 2i + 1) are rotated by row
    positions[t] (int32 [T]; default: row t); a position outside the table gives NaN.

    Values are rounded once, from fp32 or better; k's codes are those of the 64-bit value
    but where a rotation leaves little of its terms or a code is subnormal.  q comes
    back in its own type (fp32 too, which paged_attention does not take).  A page's scale is the least power of
    two that holds its new values within 448 (a non-finite one is stored as NaN and
    does not count); if the page already holds tokens, the scale never falls, and where it
    grows their codes are rounded again.  The pages that a call appends to must be
    distinct."""
    r = (_lib._paged_host or _lib.paged_host()).append_kv(
        pages, k, v, page_table, lengths, cu_tokens, freqs_cis, positions, k_weight, q, q_weight,
        eps)
    if r is not None:
        return None if r is True else r
    name = "append_kv"
    T = k.shape[0]
    H, D = _check_cache(name, pages, page_table, lengths, cu_tokens, T)
    _check_rows(name, k, H, D, "k")
    _check_rows(name, v, H, D, "v")
    _check(v.shape[0] == T, f"{name}: k has {T} rows, v {v.shape[0]}")
    dt = _lib.dtype_code(k, "k")
    _lib.require_dtype(v, k.dtype, "v")
    if q is not None:
        _check_rows(name, q, None, D, "q")
        _check(q.shape[0] == T and q.shape[1] > 0, f"{name}: k has {T} rows, q {tuple(q.shape)}")
        _lib.require_dtype(q, k.dtype, "q")
    _check(q is not None or q_weight is None, f"{name}: q_weight without q")
    _check(freqs_cis is not None or positions is None, f"{name}: positions without freqs_cis")
    kn = _norm(name, k_weight, H, D, "k_weight")
    qn = _norm(name, q_weight, q.shape[1] if q is not None else 0, D, "q_weight")
    wt = _lib.DT_BF16
    for w, n in ((k_weight, "k_weight"), (q_weight, "q_weight")):
        if w is not None:
            wt = _lib.dtype_code(w, n)
    if kn and qn:
        _lib.require_dtype(q_weight, k_weight.dtype, "q_weight")
    cs = None
    if freqs_cis is not None:
        _check(torch.is_complex(freqs_cis) and freqs_cis.shape[-1] == D // 2,
               f"{name}: freqs_cis must be complex [rows, {D // 2}]")
        cs = _rotations(freqs_cis)
        if positions is None:
            _check(cs.shape[0] >= T, f"{name}: freqs_cis has {cs.shape[0]} rows for {T} tokens")
        else:
            _lib.require_dtype(positions, torch.int32, "positions")
            _check(tuple(positions.shape) == (T,) and positions.is_contiguous(),
                   f"{name}: positions must be a contiguous [{T}]")
            _check(cs.shape[0] > 0, f"{name}: freqs_cis is empty")
    _one_device(name, *pages, k, v, q, page_table, lengths, cu_tokens, cs, positions, k_weight,
                q_weight)
    with torch.cuda.device(k.device):
        k, v = _aligned(k), _aligned(v)
        q = None if q is None else _aligned(q)
        kw = None if k_weight is None else _aligned(k_weight.reshape(-1))
        qw = None if q_weight is None else _aligned(q_weight.reshape(-1))
        cs = None if cs is None else _aligned(cs)
        out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        L = _lib.lib()
        n = L.fvsr_kv_append_workspace_floats(T, kn)
        ws = torch.empty(n, dtype=torch.float32, device=k.device) if n else None
        _lib.check(L.fvsr_kv_append(
            ctypes.byref(_cache_arg(pages, page_table, lengths, cu_tokens)), k.data_ptr(),
            k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _lib.ptr(q),
            0 if q is None else q.stride(0), 0 if q is None else q.stride(1),
            0 if q is None else q.shape[1], _lib.ptr(out), dt, T, _lib.ptr(kw), kn, _lib.ptr(qw),
            qn, wt, float(eps), _lib.ptr(cs), 0 if cs is None else cs.shape[0],
            _lib.ptr(positions), _lib.ptr(ws), n, _lib.stream(k)), name)
    return out


def paged_attention(q: torch.Tensor, pages: KVPages, page_table: torch.Tensor,
                    lengths: torch.Tensor, cu_tokens: torch.Tensor | None = None, *,
                    causal: bool = True, keep: torch.Tensor | None = None,
                    sm_scale: float | None = None, out: torch.Tensor | None = None):
    """softmax(q k^T * sm_scale) v over each sequence's pages.

    q [T, q_heads, head_dim] bf16 or fp16, q_heads a multiple of the cache's
    heads (head h reads key/value head h // (q_heads // heads)); rows may be
    strided.  The n rows of sequence b are its last n positions, lengths[b] - n and
    on (lengths as in append_kv: tokens of this step included).  causal: a row
    sees the positions up to its own; otherwise every token of its sequence.
    keep: bool [q_heads, NQ, NK], or [B, q_heads, NQ, NK]: queries 128 i .. 128
    i + 127 of a sequence's rows see its page j only where keep[..., i, j]; blocks outside
    the mask are not kept.  sm_scale: 1 / sqrt(head_dim) by default, positive.

    Returns out, or a new tensor like q.  A row that sees nothing is zero; rows
    behind cu_tokens[B] are zero in a new tensor and left alone in a given one.  A page
    id outside the pool makes the rows that read it NaN; what a mask hides, or lies
    behind a length, does not count even if it is NaN.  Logits and sums are fp32
    accumulators of the matrix cores, which keep a sum to 2^-12 of its terms' magnitudes (2^-15
    on Gaussian values): a logit is off by as much of sm_scale * sum |q k|.  The weights
    count with q's precision (2^-8 or 2^-12) or 2^-22 of the largest."""
    if out is None:
        r = (_lib._paged_host or _lib.paged_host()).paged_attention(
            q, pages, page_table, lengths, cu_tokens, causal, keep, sm_scale)
        if r is not None:
            return r
    name = "paged_attention"
    _check(q.dim() == 3, f"{name}: q must be [T, heads, head_dim], got {tuple(q.shape)}")
    T, Hq = q.shape[:2]
    H, D = _check_cache(name, pages, page_table, lengths, cu_tokens, T)
    _check_rows(name, q, None, D, "q")
    _check(Hq > 0 and Hq % H == 0, f"{name}: {Hq} query heads over {H} key/value heads")
    dt = _lib.dtype_code(q, "q")
    if dt == _lib.DT_F32:
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    _check(0.0 < scale < 3e38, f"{name}: sm_scale must be positive, got {scale}")
    nq = nk = 0
    if keep is not None:
        B = page_table.shape[0]
        _lib.require_dtype(keep, torch.bool, "keep")
        if keep.dim() == 3 and B == 1:
            keep = keep[None]
        _check(keep.dim() == 4 and keep.shape[:2] == (B, Hq),
               f"{name}: keep must be [{B}, {Hq}, query blocks, pages], got {tuple(keep.shape)}")
        if keep.numel() == 0:  # nothing is kept
            keep = keep.new_zeros((B, Hq, 1, 1))
        nq, nk = keep.shape[2:]
    fresh = out is None
    if not fresh:
        _lib.require_dtype(out, q.dtype, "out")
        _check(out.shape == q.shape and out.stride(2) == 1 and out.stride(0) % 4 == 0 and
               out.stride(1) % 4 == 0 and out.data_ptr() % 8 == 0 and
               all(n == 1 or s > 0 for n, s in zip(out.shape, out.stride())),
               f"{name}: out must be {tuple(q.shape)} with 8-byte aligned rows of their own")
    _one_device(name, q, *pages, page_table, lengths, cu_tokens, keep, out)
    with torch.cuda.device(q.device):
        q = _aligned(q)
        keep = None if keep is None else keep.contiguous()
        if fresh:
            out = (torch.empty if page_table.shape[0] else torch.zeros)(
                q.shape, dtype=q.dtype, device=q.device)
        L = _lib.lib()
        cache = ctypes.byref(_cache_arg(pages, page_table, lengths, cu_tokens))
        n = L.fvsr_paged_attn_workspace_floats(cache, T, Hq, int(keep is not None))
        ws = torch.empty(n, dtype=torch.float32, device=q.device) if n else None
        _lib.check(L.fvsr_paged_attn(
            cache, q.data_ptr(), q.stride(0), q.stride(1), Hq, out.data_ptr(), out.stride(0),
            out.stride(1), dt, T, int(bool(causal)), _lib.ptr(keep), nq, nk, scale, int(fresh),
            _lib.ptr(ws), n, _lib.stream(q)), name)
    return out
