"""Drawing tokens on the device: temperature, top-k, top-p and min-p from given random numbers.

``generate.generate_fast`` filters and draws one sentence's tokens with the reference's own torch
operations, whose random stream it follows.  Programs that run several sequences draw all of
their next tokens in one call here, each row with settings of its own, and nothing waits for the
device.  The random numbers are an input (``torch.rand(rows, device=...)``, or what a request's own
generator gives), so the same numbers draw the same tokens in an eager call, a replayed graph, and
whatever other rows the call holds::

    u.uniform_(generator=g)
    token, logprob = sampling.sample(logits, u, temperature, top_k=50, top_p=0.9,
                                     return_logprob=True)

``RuntimeError`` for a wrong shape, type or device.
"""
from __future__ import annotations

import torch

from . import ops


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: float | torch.Tensor = 1.0,
           top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0,
           min_p: float | torch.Tensor = 0.0, return_logprob: bool = False):
    """int64 ``[rows]``: a token of each row of ``logits [rows, vocab]`` (bf16, fp16 or fp32, vocab
    at most 2^20; ``mtl_sample``), drawn with ``u`` fp32 ``[rows]`` in [0, 1).

    A row's tokens stand in an order: the larger logit first, of equal ones the lower index.  With
    w_i = exp((x_i - max x) / temperature), the first ``top_k`` of the order stay (0: all); of
    these, those before which weights of at most ``top_p`` times these' sum lie (1: all); of these,
    those of w_i >= ``min_p``.  The first of the order always stays.  The token is the lowest index
    at which the weights of those that stay, summed by index, exceed u times their sum.

    Each setting is a number or a tensor ``[rows]`` (fp32, ``top_k`` int32).  A temperature that is
    not above 0 takes the first of the order.  NaN logits count as -infinity and are never drawn; a
    row of nothing else gives -1.  Weights are of 64 bits and summed as the nearest multiples of
    2^-n, n = 51 up to 4096 tokens and one less for each doubling (45 for 151 936): a token of less
    than half of that is not drawn.  With ``return_logprob`` also the fp32 logarithm of the token's
    probability among those that stayed (0 without temperature, -infinity for -1).  An expanded row
    of logits draws several tokens from it."""
    t, k, p, m = (x if isinstance(x, torch.Tensor) else None
                  for x in (temperature, top_k, top_p, min_p))
    op = ops.overload("sample_logprob" if return_logprob else "sample")
    return op(logits, u, t, k, p, m, 1.0 if t is not None else float(temperature),
              0 if k is not None else int(top_k), 1.0 if p is not None else float(top_p),
              0.0 if m is not None else float(min_p))
