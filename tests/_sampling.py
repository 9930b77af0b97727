"""The draw of a token from its definition, one row at a time in float64 on the host."""
import math

import numpy as np
import torch


def order_of(x):
    """Larger logits first, of equal ones the lower index (NaN as -infinity)."""
    x = np.where(np.isnan(x), -np.inf, x)
    return x, np.argsort(-x, kind="stable")


def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob, the sums' distance to the nearest border as a part of the whole)."""
    x, order = order_of(np.asarray(x, dtype=np.float64))
    if x[order[0]] == -np.inf:
        return -1, -math.inf, 1.0
    f = [float(np.float32(z)) for z in (temperature, top_p, min_p)]
    t, p, m = f
    if not t > 0:
        return int(order[0]), 0.0, 1.0
    top = x[order[0]]
    if 0 < top_k < len(order):
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t))
    w[np.isnan(w)] = 0.0
    total = math.fsum(w)
    before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
    keep = w > 0
    near = 1.0
    if p < 1:
        keep &= before <= p * total
        near = min(near, np.abs(before[1:] - p * total).min(initial=total) / total)
    keep &= w >= m
    if m > 0 and (w != 1).any():                     # the largest logits' weight is 1 exactly
        near = min(near, np.abs(w[w != 1] / m - 1).min())
    keep[0] = True
    pairs = sorted((int(i), float(v)) for i, v in zip(order[keep], w[keep]))
    c = np.cumsum([v for _, v in pairs])
    goal = float(np.float32(u)) * c[-1]
    j = min(int(np.searchsorted(c, goal, side="right")), len(pairs) - 1)
    near = min(near, np.abs(c - goal).min() / c[-1])
    return pairs[j][0], math.log(pairs[j][1] / c[-1]), near


def reference(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = logits.shape[0]
    x, u = logits.detach().cpu().double().numpy(), u.cpu().tolist()
    s = [z.tolist() if isinstance(z, torch.Tensor) else [z] * rows
         for z in (temperature, top_k, top_p, min_p)]
    return [draw(x[r], u[r], *(z[r] for z in s)) for r in range(rows)]
