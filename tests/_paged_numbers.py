"""Attention inputs whose outputs are known in closed form, and a check that allows nothing but the
output's own rounding and float32 sums: for errors that an allowance for random inputs would
hide."""
import torch

from tests._paged import TYPES, table_for

DIM0 = 16               # levels of the scores: position p has level (p % DIM0) / DIM0


def spread_pages(rows_k, rows_v, lens, Hkv, page, kv, gen, spare=2, width=0):
    """Rows [n, dim] a sequence into shuffled pages; what no sequence holds is NaN."""
    width = max([width, 1] + [-(-n // page) for n in lens])
    pages = sum(-(-n // page) for n in lens) + spare
    table = table_for(lens, page, width, pages, gen)
    pools = []
    for rows in (rows_k, rows_v):
        pool = torch.full((pages, Hkv, page, rows[0].shape[1]), float("nan"), dtype=TYPES[kv])
        for i, n in enumerate(lens):
            for j in range(-(-n // page)):
                part = rows[i][j * page:min(n, (j + 1) * page)]
                assert torch.equal(part.to(TYPES[kv]).double(), part)      # exact in the type
                pool.view(torch.uint8 if kv == "e4m3" else pool.dtype)[
                    int(table[i, j]), :, :len(part)] = part.to(TYPES[kv]).view(
                        torch.uint8 if kv == "e4m3" else pool.dtype)
        pools.append(pool)
    return (*pools, table)


def heads_of(B, H, D, typ):
    """Queries that read dim 0 with a factor of their own: 1, 1 1/8, ... 1 7/8."""
    q = torch.zeros(B, H, D, dtype=torch.float64)
    q[:, :, 0] = 1 + torch.arange(H).double() % 8 / 8
    return q.to(TYPES[typ])


def coded_case(lens, H, Hkv, D, page, typ, kv, code, c=2.0, seed=0, width=0):
    """Scores by (position % 16), V one-hot by position or by tile of 32 positions: out[d] is the
    weight of the positions with code d.  -> (arguments, what each head attends with)"""
    gen = torch.Generator().manual_seed(seed)
    k, v = [], []
    for n in lens:
        p = torch.arange(n)
        x = torch.zeros(n, D, dtype=torch.float64)
        x[:, 0] = (p % DIM0).double() / DIM0
        k.append(x)
        at = (p if code == "position" else p // 32) % D
        v.append(torch.nn.functional.one_hot(at, D).double())
    kp, vp, table = spread_pages(k, v, lens, Hkv, page, kv, gen, width=width)
    q = heads_of(len(lens), H, D, typ)
    args = dict(q=q, k_pages=kp, v_pages=vp, table=table,
                lens=torch.tensor(lens, dtype=torch.int32), scale=c)
    return args, closed_form(q, k, v, c)


def sink_case(lens, H, Hkv, D, page, typ, kv, c, seed=0, width=0):
    """Position 0 scores c to 1.875 c above all others and has V = 0: the output is the others'
    share, which is as small as their weight.  V is large, so that it is no subnormal number."""
    gen = torch.Generator().manual_seed(seed)
    k, v = [], []
    for n in lens:
        x = torch.zeros(n, D, dtype=torch.float64)
        x[:1, 0] = 1
        k.append(x)
        y = (128 * (1 + torch.arange(D).double() % 8 / 8)).repeat(n, 1)
        y[:1] = 0
        v.append(y)
    kp, vp, table = spread_pages(k, v, lens, Hkv, page, kv, gen, width=width)
    q = heads_of(len(lens), H, D, typ)
    args = dict(q=q, k_pages=kp, v_pages=vp, table=table,
                lens=torch.tensor(lens, dtype=torch.int32), scale=c)
    return args, closed_form(q, k, v, c)


def closed_form(q, k, v, c, weights=lambda w: w):
    """(out, lse) in float64; `weights` for planted mistakes."""
    q = q.double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64)
    for i, (x, y) in enumerate(zip(k, v)):
        if len(x) == 0:
            continue
        s = q[i] @ x.T * c
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - top)
        total = w.sum(-1, keepdim=True)
        out[i] = weights(w) @ y / total
        lse[i] = (top + torch.log(total))[:, 0]
    return out, lse


def room(n, typ, drop=0.0):
    """The relative error of sum w v / sum w for V of one sign, n positions, the smallest weight
    e^-drop of the largest.  Twice, for numerator and sum: sums of n terms in float32 (2^-24 a
    term), exp2 and the score's own roundings (|s| 2^-22, |s| at most drop + 8).  Once: the weights'
    two terms (bf16: 2^-8 of 2^-8; f16, cut: 2^-10 of 2^-10, and 2^-39 of the largest weight)."""
    terms = 2.0 ** -16 if typ == "bf16" else 2.0 ** -20 + 2.0 ** -39 * 2.718281828 ** drop
    return 2 * (n * 2.0 ** -24 + (drop + 8) * 2.0 ** -22 + 2.0 ** -22) + terms


def beside(got, ref, rel):
    """Where got is not what a value within rel of ref rounds to in got's type."""
    t = got.dtype
    lo, hi = ((ref * (1 - s * rel)).to(t).double() for s in (1, -1))
    x = got.double()
    return ~((torch.minimum(lo, hi) <= x) & (x <= torch.maximum(lo, hi)))
