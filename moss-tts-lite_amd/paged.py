"""Paged key-value cache: many sequences in one pool of pages on the device.

The decoder's own cache (``model.Int4Backbone``) is dense and holds one sequence, as the
reference's does (moss_tts_lite/model.py:110-112).  Programs that run several sequences at once
(candidates of one sentence, requests of a server) keep their keys and values in pages instead:

* ``k_pages``, ``v_pages``: ``[layers, pages, kv_heads, page_size, head_dim]`` in bfloat16,
  float16 or float8_e4m3fn (a stored element times its kv head's ``k_scale`` / ``v_scale`` is
  the value).  The attention and the write take one layer ``[pages, kv_heads, page_size,
  head_dim]``; its strides are free as long as ``head_dim`` is adjacent and rows are 16-byte
  aligned, so ``[pages, page_size, kv_heads, head_dim]`` memory is passed as a transposed view.
  page_size 16, 32, 64, 128 or 256; head_dim 64 or 128.
* ``table`` int32 ``[seqs, width]``: the pages of each sequence, in the order of its positions.
  An entry outside the pool (-1 where a sequence holds no page) is a hole: its positions take
  no part in the attention and are not written.
* ``lens`` int32 ``[seqs]``: tokens of each sequence; it holds ``ceil(len / page_size)`` pages.
* ``refs`` int32 ``[pages]``: how many sequences hold a page; 0 is a free page.

Everything lives and is decided on the device, nothing waits for it, every launch goes to the
current stream and can be captured into a graph.  The bookkeeping calls return a ``status``
tensor (0 done, 1 not enough free pages, 2 a bad argument), and one that is not 0 has changed
nothing; :func:`check` reads it and raises.  ``RuntimeError`` for a wrong shape, type or device.

After a refused :func:`pages_extend` the lengths are the old ones, and the position before a
sequence's end is a token that is there already, on a page that others may hold too.  A loop that
does not wait for the status makes its rows padding then.  One token of every sequence in ``seqs``::

    status = paged.pages_extend(table, lens, refs, seqs, torch.ones_like(seqs), k, v)
    rows, n = table[seqs], lens[seqs]
    at = torch.where(status == 0, n.long() - 1, -1)
    for l in range(layers):
        q = paged.paged_write(qkv[l], k[l], v[l], rows, at, None, q_norm, k_norm, cos, sin)
        out = paged.paged_attention(q, k[l], v[l], rows, n, scale)
"""
from __future__ import annotations

import torch

from . import ops


def new_cache(layers: int, pages: int, kv_heads: int, page_size: int, head_dim: int, seqs: int,
              width: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
    """Empty ``(k_pages, v_pages, table, lens, refs)`` for ``seqs`` sequences of at most
    ``width`` pages each."""
    shape = (layers, pages, kv_heads, page_size, head_dim)
    return (torch.zeros(shape, dtype=dtype, device=device),
            torch.zeros(shape, dtype=dtype, device=device),
            torch.full((seqs, width), -1, dtype=torch.int32, device=device),
            torch.zeros(seqs, dtype=torch.int32, device=device),
            torch.zeros(pages, dtype=torch.int32, device=device))


def check(status: torch.Tensor) -> None:
    """Waits for a bookkeeping call's ``status`` and raises ``RuntimeError`` unless it is 0."""
    code = int(status)
    if code == 1:
        raise RuntimeError("not enough free pages")
    if code:
        raise RuntimeError("a sequence index out of range or given twice, or a length that does "
                           "not fit")


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    table: torch.Tensor, lens: torch.Tensor, scale: float,
                    k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    return_lse: bool = False):
    """Attention of one query token of each sequence over its pages (``mtl_paged_attention``):
    ``q [seqs, heads, head_dim]`` bf16 or fp16, any strides; softmax and sums in fp32.  Returns
    ``out`` like q, and with ``return_lse`` also the fp32 ``[seqs, heads]`` logarithm of the
    softmax sums, with which the result joins that of other keys.  A sequence without positions
    gives 0 and -inf.  Lengths past the table's width count as that width.  The same call gives
    the same bits; the order of a sequence's sums goes by all lengths of the call.  What lies in
    a hole or past a length has no effect, NaN included; K and V of the positions attended to
    are finite (an infinity or NaN there gives NaN where it enters)."""
    op = ops.overload("paged_attention_lse" if return_lse else "paged_attention")
    return op(q, k_pages, v_pages, table, lens, scale, k_scale, v_scale)


def paged_attention_shared(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           table: torch.Tensor, lens: torch.Tensor, groups: torch.Tensor,
                           shared: torch.Tensor, scale: float,
                           k_scale: torch.Tensor | None = None,
                           v_scale: torch.Tensor | None = None, return_lse: bool = False):
    """:func:`paged_attention` for sequences that share a prefix, read once for each 64 query heads
    of a kv head (``mtl_paged_attention_shared``): forks of one sequence, requests on one prompt.
    It pays where all sequences together have some 20 000 to 40 000 shared positions (8 kv heads of
    128); below, and with 64 or more query heads to a kv head, :func:`paged_attention` is faster.

    Sequences ``groups[g]`` to ``groups[g + 1] - 1`` (int32 ``[n + 1]``, ascending from 0 to the
    number of sequences; where it does not ascend, each sequence is by itself) are a group, and its first ``shared[g]`` positions (int32 ``[n]``) lie in
    the same pages for all of them, or in copies of these: a page that :func:`pages_extend` copied
    holds the same K and V up to where the fork was made.  They are read through the table row of
    the group's first sequence that reaches them all, or, where that is faster, through each
    sequence's own.  Shorter and empty sequences of a group
    attend to what their length holds.  Results are those of :func:`paged_attention`, with sums in
    another order, and the same call gives the same bits.  K and V that any sequence of a group
    attends to are finite (an infinity or NaN there may give NaN in all of the group)."""
    op = ops.overload("paged_attention_shared_lse" if return_lse else "paged_attention_shared")
    return op(q, k_pages, v_pages, table, lens, groups, shared, scale, k_scale, v_scale)


def paged_write(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                table: torch.Tensor, positions: torch.Tensor, seqs: torch.Tensor | None = None,
                q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                eps: float = 1e-6, k_scale: torch.Tensor | None = None,
                v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """q/k RMSNorm, RoPE and the page write of new tokens (``mtl_paged_write``): row r of
    ``qkv [rows, (heads + 2 kv_heads) * head_dim]`` is position ``positions[r]`` (int64) of
    sequence ``seqs[r]`` (int32; None: sequence r), written into one layer's pages in place.
    Returns the normed, rotated ``q [rows, heads, head_dim]``.

    ``cos``, ``sin``: ``[positions, head_dim]`` tables as ``model.rope_tables`` makes them, or
    the same in float32; without norm weights or tables that step is left out.  Computed in fp32
    and rounded once (the dense decoder's kernels round after every step, as the reference
    does).  A row with a negative position, or one past the tables, is padding: q 0, nothing
    written.  No two rows may name the same position of one sequence, ``k_pages`` and ``v_pages``
    share no memory, and a page that several sequences hold is not to be written:
    :func:`pages_extend` copies it first."""
    return ops.overload("paged_write")(qkv, k_pages, v_pages, table, positions, seqs, q_norm,
                                       k_norm, cos, sin, eps, k_scale, v_scale)


def pages_extend(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, seqs: torch.Tensor,
                 counts: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor
                 ) -> torch.Tensor:
    """Room for ``counts[i]`` more tokens of sequence ``seqs[i]`` (int32 ``[n]``, n <= 1024, no
    sequence twice), in call order (``mtl_pages_extend``): a partly filled last page that other
    sequences hold too is first replaced by a copy, in all layers; then the lowest free pages are
    taken one after the other.  ``lens`` grows by ``counts``.  Returns the status; unless it is 0
    there is no room, and the last positions of the sequences are not to be written."""
    return ops.overload("pages_extend")(table, lens, refs, seqs, counts, k_pages, v_pages)


def pages_fork(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor,
               children: torch.Tensor, page_size: int) -> torch.Tensor:
    """Sequence ``children[i]`` becomes ``parents[i]``: the same pages and length, nothing is
    copied (``mtl_pages_fork``).  Children are distinct, empty and no parents.  Returns the
    status."""
    return ops.overload("pages_fork")(table, lens, refs, parents, children, page_size)


def pages_truncate(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
                   seqs: torch.Tensor, new_lens: torch.Tensor, page_size: int) -> torch.Tensor:
    """Sequence ``seqs[i]`` keeps its first ``new_lens[i]`` tokens, 0 frees it
    (``mtl_pages_truncate``); pages that no sequence holds any more are free.  Returns the
    status."""
    return ops.overload("pages_truncate")(table, lens, refs, seqs, new_lens, page_size)


def pages_compact(table: torch.Tensor, refs: torch.Tensor, k_pages: torch.Tensor,
                  v_pages: torch.Tensor):
    """Moves the held pages to the low end of the pool, in all layers (``mtl_pages_compact``,
    ``mtl_pages_copy``): with L pages held, the k-th held page at or past L goes to the k-th free
    page below L.  Returns new ``(table, refs, live)`` with ``live`` int32 ``[1]`` = L; the pages
    at and past it are free.  The old table and counts stay as they are, and valid until a page
    is next taken or written."""
    return ops.overload("pages_compact")(table, refs, k_pages, v_pages)


def pages_copy(k_pages: torch.Tensor, v_pages: torch.Tensor, src: torch.Tensor,
               dst: torch.Tensor) -> None:
    """Copies page ``src[i]`` onto page ``dst[i]`` (int32 ``[n]``) in every layer
    (``mtl_pages_copy``).  Pairs outside the pool are skipped; no page may be ``dst`` twice or
    both a source and a destination."""
    ops.overload("pages_copy")(k_pages, v_pages, src, dst)
