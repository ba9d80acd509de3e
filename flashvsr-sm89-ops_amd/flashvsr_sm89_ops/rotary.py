"""Rotary positions for q and k, forward and backward, on gfx950.

The reference rotates interleaved pairs of the whole head by a table of complex numbers, behind
an RMSNorm (flashvsr_sm89_ops/fused_rms_rope.py:66-83).  `rotary` is for what lies beside
that: halves or interleaved pairs, part of the head, frequencies stretched for long contexts,
any positions without a table, and training.

    freqs = rotary_frequencies(128, base=500000.0, scaling="parts", factor=8.0, context=8192)
    q, k = rotary(q, k, freqs, positions)
    append_kv(pages, k, v, table, lengths)
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib

_PAIRS = {"half": _lib.PAIRS_HALF, "interleaved": _lib.PAIRS_INTERLEAVED}


class RotaryFrequencies(NamedTuple):
    """Pair i turns by position * turns[i] (1 is a whole turn); results are scaled by gain."""
    turns: torch.Tensor  # [channels / 2] float64
    gain: float = 1.0


def rotary_frequencies(channels: int, base: float = 10000.0, *, scaling: str | None = None,
                       factor: float = 1.0, context: int | None = None, fast: float = 32.0,
                       slow: float = 1.0, gain: float | None = None,
                       device="cuda") -> RotaryFrequencies:
    """Frequencies base^(-2 i / channels), i = 0 .. channels / 2 - 1, of the first `channels`
    channels of a head, and how they are stretched for a context `factor` times the one that a
    model was trained on:

    scaling None      as they are
            "linear"  all divided by the factor (positions are squeezed)
            "base"    a base of base * factor^(channels / (channels - 2)): the fastest pair stays,
                      the slowest is divided by the factor
            "parts"   pairs that turn `fast` times or more over `context` tokens (the old length)
                      stay, those that turn `slow` times or less are divided by the factor,
                      linear in the turns between.  (A model that was trained with another ramp,
                      such as one linear in i between two rounded pairs, needs its own: a
                      RotaryFrequencies of `turns` made by hand.)

    gain: what q and k are scaled by; by default 0.1 ln(factor) + 1 with "parts", else 1."""
    def need(ok, what):
        if not ok:
            raise ValueError(f"rotary_frequencies: {what}")
    need(channels > 0 and channels % 2 == 0, f"channels must be even and positive, got {channels}")
    need(0.0 < base < math.inf, f"base must be positive, got {base}")
    need(1.0 <= factor < math.inf, f"factor must be 1 or more, got {factor}")
    need(scaling in (None, "linear", "base", "parts"), f"unknown scaling {scaling!r}")
    need(scaling is not None or factor == 1.0, f"factor {factor} without scaling")
    if scaling == "base":
        need(channels > 2, "scaling 'base' needs more than 2 channels")
        base = base * factor ** (channels / (channels - 2))
    inv = base ** (-torch.arange(0, channels, 2, dtype=torch.float64) / channels)
    if scaling == "linear":
        inv = inv / factor
    if scaling == "parts":
        need(context is not None and context > 0, "scaling 'parts' needs the old context")
        need(0.0 <= slow < fast < math.inf, f"slow {slow} must be below fast {fast}")
        keep = ((context * inv / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        inv = keep * inv + (1.0 - keep) * inv / factor
    if gain is None:
        gain = 0.1 * math.log(factor) + 1.0 if scaling == "parts" else 1.0
    need(math.isfinite(gain), f"gain must be finite, got {gain}")
    return RotaryFrequencies((inv / (2 * math.pi)).to(device), float(gain))


class _Rows(ctypes.Structure):
    """fvsr_rotary_rows."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "y")] +
                [(n, ctypes.c_int64) for n in ("heads", "x_batch", "x_tok", "x_head")])


def _launch(xs, turns, gain, positions, pairs, back):
    """Each of xs [B, S, heads, head_dim] turned, in new tensors."""
    B, S, _, D = xs[0].shape
    with torch.cuda.device(xs[0].device):
        # (A gradient may be one value spread over a shape.)
        xs = [x if x.stride(3) == 1 or D == 1 else x.contiguous() for x in xs]
        ys = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs]
        rows = [_Rows(x.data_ptr(), y.data_ptr(), x.shape[2], *x.stride()[:3])
                for x, y in zip(xs, ys)]
        _lib.check(_lib.lib().fvsr_rotary(
            ctypes.byref(rows[0]), ctypes.byref(rows[1]) if len(rows) > 1 else None,
            _lib.dtype_code(xs[0], "q"), B, S, D, 2 * turns.numel(), turns.data_ptr(),
            _lib.ptr(positions), 0 if positions is None or positions.dim() == 1 else
            positions.stride(0), gain, pairs, int(back), _lib.stream(xs[0])), "rotary")
    return ys


_ELSEWHERE = ("rotary: a leaf of a captured step still has a graph from another stream: let go of "
              "its outputs first, or capture with leaves of its own")


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, turns, gain, positions, pairs, back, *xs):
        ctx.save_for_backward(turns, positions)
        ctx.how = gain, pairs, back
        return tuple(_launch(xs, turns, gain, positions, pairs, back))

    @staticmethod
    def backward(ctx, *grads):
        if _lib.host().graph_behind():
            raise RuntimeError(_ELSEWHERE if _lib.host() is not _lib._GeneralPath else
                               "rotary: a backward pass is captured with the native extension only")
        turns, positions = ctx.saved_tensors
        gain, pairs, back = ctx.how
        # The transpose of a rotation is the one back; the gain stays.
        return (None,) * 5 + _Rotary.apply(turns, gain, positions, pairs, not back, *grads)


def rotary(q: torch.Tensor, k: torch.Tensor | None, freqs: RotaryFrequencies,
           positions: torch.Tensor | None = None, *, pairs: str = "half"):
    """q and k with their positions: (q, k), or q alone without a k, in new tensors.

    q [T, heads, head_dim] or [B, S, heads, head_dim], k the same with heads of its own; bf16,
    fp16 or fp32, both of one type; rows may be strided (columns of a fused qkv).  The first
    2 * len(freqs.turns) channels of each head are rotated, pairs "half": (i, i + n / 2) of those n,
    "interleaved": (2 i, 2 i + 1); the others are copied.

    positions int32, [T] or [S] (the same for all B) or [B, S]; default: 0, 1, ..  Whole turns
    are taken off position * turns in 64 bits; sines, products and sums are fp32, rounded once.

    Differentiable in q and k (any number of times, backward mode); freqs and positions have no
    gradient.  A step with its backward pass captures into a graph where its leaves have no
    graph from outside the capture left: an earlier step's outputs are let go first.  Otherwise the
    backward pass is refused, for leaves further up too, and in a capture so is a call that is given
    such a leaf itself, unless under no_grad.  Without the native extension no backward pass is
    captured."""
    r = (_lib._selected_host or _lib.selected_host()).rotary(q, k, freqs, positions, pairs)
    if r is not None:
        return r
    name = "rotary"

    def check(ok, what):
        if not ok:
            raise ValueError(f"{name}: {what}")
    check(q.dim() in (3, 4), f"q must be [T, heads, head_dim] or [B, S, heads, head_dim], got "
          f"{tuple(q.shape)}")
    check(k is None or (k.dim() == q.dim() and k.shape[:-2] == q.shape[:-2] and
                        k.shape[-1] == q.shape[-1]),
          f"k must be {tuple(q.shape[:-2])} x heads x {q.shape[-1]}, got "
          f"{None if k is None else tuple(k.shape)}")
    _lib.dtype_code(q, "q")
    if k is not None:
        _lib.require_dtype(k, q.dtype, "k")
    if pairs not in _PAIRS:
        raise ValueError(f"{name}: pairs must be 'half' or 'interleaved', got {pairs!r}")
    turns, gain = freqs
    _lib.require_dtype(turns, torch.float64, "freqs.turns")
    check(turns.dim() == 1 and turns.is_contiguous() and 2 * turns.numel() <= q.shape[-1],
          f"freqs.turns must be a contiguous vector for at most {q.shape[-1]} channels, got "
          f"{tuple(turns.shape)}")
    check(not turns.requires_grad, "freqs have no gradient")
    lead = q.shape[:-2]
    if positions is not None:
        _lib.require_dtype(positions, torch.int32, "positions")
        check(positions.shape in (lead, lead[-1:]) and (positions.shape[-1] <= 1 or
                                                        positions.stride(-1) == 1),
              f"positions must be {tuple(lead[-1:])} or {tuple(lead)} with unit-stride rows, got "
              f"{tuple(positions.shape)}")
    xs = [x for x in (q, k) if x is not None]
    _lib.require_gpu(*xs, turns, positions)
    check(all(t is None or t.device == q.device for t in (k, turns, positions)),
          "tensors on several devices")
    check(all(unpack_dual(x).tangent is None for x in xs), "no forward-mode gradients")
    four = [x if x.dim() == 4 else x[None] for x in xs]
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        if any(_lib.host().graph_elsewhere(x) for x in xs):
            raise RuntimeError(_ELSEWHERE)
        ys = _Rotary.apply(turns, float(gain), positions, _PAIRS[pairs], False, *four)
    else:
        ys = _launch(four, turns, float(gain), positions, _PAIRS[pairs], False)
    ys = [y if q.dim() == 4 else y[0] for y in ys]
    return ys[0] if k is None else (ys[0], ys[1])
