"""Rotation of queries and keys by their positions, with the RMSNorm of each head in the same pass.

The decoder's own step rotates whole heads, half against half, out of a bf16 table of its cache's
length (``model.rope_tables``, ``fast.py``).  ``paged.paged_write`` takes such tables too, and where
they do (whole heads, half against half, any frequencies, a row for each position) it norms, rotates
and writes in one launch, which is the faster way: 16 rows 2.9 us against 6.1 for the two launches
below.  This is for what tables do not give: other layouts, part of a head, positions of which no
table is held.

Rows that go into a paged cache are rotated where they lie, in the q | k | v matrix, and then
written as they are::

    q, k, _ = qkv.split([heads * d, kv_heads * d, kv_heads * d], 1)
    rotary.qk_rotary_(q.unflatten(1, (heads, d)), k.unflatten(1, (kv_heads, d)), positions, freqs,
                      q_norm, k_norm)
    q = paged.paged_write(qkv, k_pages, v_pages, rows, positions)

``RuntimeError`` for a wrong shape, type or device.
"""
from __future__ import annotations

import math

import torch

from . import ops


def rotary_freqs(turned: int, base: float = 10000.0, factor: float = 1.0,
                 original: int | None = None, slow: float = 1.0, fast: float = 32.0,
                 device="cuda", ramp: str = "dims") -> torch.Tensor:
    """float64 ``[turned / 2]`` frequencies in radians a position: f_t = base^(-2t / turned).

    ``factor`` > 1 stretches them for contexts ``factor`` times as long.  Without ``original``
    every frequency is divided by it (positions are interpolated).  With ``original``, the context
    a model was trained on, a dim that makes ``fast`` turns or more within it keeps its frequency,
    one that makes ``slow`` turns or fewer is divided by ``factor``, and in between it gets
    (1 - g) f_t / factor + g f_t.  g falls from 1 to 0

    * with ``ramp="dims"`` evenly from dim to dim, where dim t makes original f_t / (2 pi) turns:
      g = (b - t) / (b - a), a (rounded down, at least 0) the dim of ``fast`` turns, b (rounded up,
      below ``turned``) that of ``slow``.  Checkpoints whose configuration has ``rope_type`` "yarn"
      (``beta_slow``, ``beta_fast``) are made for this, with :func:`rotary_amplitude`;
    * with ``ramp="turns"`` with the number n of turns: g = (n - slow) / (fast - slow).  This is for
      configurations that give ``low_freq_factor`` and ``high_freq_factor`` (here ``slow`` and
      ``fast``), with amplitude 1.

    Raising the base instead, by factor^(turned / (turned - 2)), is a matter of ``base``."""
    if turned < 0 or turned % 2:
        raise RuntimeError(f"turned must be even, got {turned}")
    if not (base > 0 and factor > 0):
        raise RuntimeError("base and factor must be positive")
    if ramp not in ("dims", "turns"):
        raise RuntimeError(f'ramp must be "dims" or "turns", got {ramp!r}')
    t = torch.arange(0, turned, 2, dtype=torch.float64)
    f = base ** (-t / max(turned, 1))
    if factor != 1.0:
        if original is None:
            f = f / factor
        else:
            if not (original > 0 and fast > slow):
                raise RuntimeError("original must be positive and fast above slow")
            if ramp == "turns":
                keep = ((original * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
            else:
                keep = _kept_by_dims(t / 2, turned, base, original, slow, fast)
            f = f / factor * (1 - keep) + f * keep
    return f.to(device)


def _kept_by_dims(t: torch.Tensor, turned: int, base: float, original: int, slow: float,
                  fast: float) -> torch.Tensor:
    """How much of dim t's own frequency stays where it falls evenly over the dims."""
    if not (base > 1 and slow > 0 and all(math.isfinite(x) for x in (base, original, fast))):
        raise RuntimeError('base must be above 1, slow above 0 and all finite for ramp="dims"')
    a, b = (turned * math.log(original / (2 * math.pi * n)) / (2 * math.log(base))
            for n in (fast, slow))
    a, b = max(math.floor(a), 0), min(math.ceil(b), turned - 1)
    if b <= 0:                                       # no dim makes more than `slow` turns
        return torch.zeros_like(t)
    return 1 - ((t - a) / max(b - a, 1)).clamp(0, 1)  # a = b: dims up to a stay


def rotary_amplitude(factor: float) -> float:
    """0.1 ln(factor) + 1 (1 up to factor 1): what cosines and sines are multiplied with where
    :func:`rotary_freqs` stretches with ``original`` and ``ramp="dims"``, so that the softmax over
    more keys stays as sharp."""
    return 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0


def qk_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor,
              q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
              eps: float = 1e-6, interleaved: bool = False, amplitude: float = 1.0):
    """``(q, k)``, each head normed (``mtl_qk_rotary``; ``q_norm``, ``k_norm`` ``[head_dim]``, or
    None: as it is) and its first ``2 * len(freqs)`` dims rotated by ``positions[row] * freqs``:
    pairs (t, t + len(freqs)), or (2t, 2t + 1) with ``interleaved``; the other dims stay.
    ``amplitude`` multiplies the rotated dims.

    ``q [rows, heads, head_dim]``, ``k [rows, kv_heads, head_dim]``: bf16 or fp16, any strides,
    head_dim a multiple of 8 up to 512.  ``positions`` int64 ``[rows]`` below 2^53, ``freqs``
    float64.  Angles are formed in 64 bits, the rest in fp32, with one rounding.  A row with a
    negative position is padding: 0."""
    return ops.overload("qk_rotary")(q, k, positions, freqs, q_norm, k_norm, eps, interleaved,
                                     amplitude)


def qk_rotary_(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
               eps: float = 1e-6, interleaved: bool = False, amplitude: float = 1.0) -> None:
    """:func:`qk_rotary` in place, for example in a q | k | v matrix.  Rows of padding stay as
    they are.  The heads of q and k must not overlap, be 16-byte aligned and have adjacent
    elements."""
    ops.overload("qk_rotary_")(q, k, positions, freqs, q_norm, k_norm, eps, interleaved, amplitude)
