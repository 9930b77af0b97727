"""What is timed of the paged key-value cache: attention of one new token a sequence over pages,
the write of new tokens into pages, branching sequences (drop, fork, extend with its copies of
shared pages) and compaction.

``listed()`` names the cases, ``draw(rng)`` gives others of the same ranges, ``prepare`` builds
what a program holds before the call (page pools, table, lengths, reference counts, rows), ``run``
is one pass: with ``own`` through the framework's entry points, else in plain torch operations in
float32.  ``exact`` computes the same from the definitions in float64 (bookkeeping: on the host,
one entry after the other), ``work`` is what a pass cannot do without.

Four kinds of case:

* ``attend``: one query token of each of ``batch`` sequences over its pages;
* ``write``: q/k RMSNorm, RoPE and the page write of a step's or a prompt's rows;
* ``branch``: the last step's candidates are dropped, their parents forked again and every
  candidate extended by a few tokens (a shared, partly filled page is copied, in all layers);
* ``compact``: the live pages of a fragmented pool move to its low end.
"""
from __future__ import annotations

import math
import random

import torch

own = False

THETA, EPS = 1_000_000.0, 1e-6
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
_E4M3_MAX = 448.0


def listed() -> list[dict]:
    return [
        # the smallest call: one sentence being spoken, a short cache
        {"name": "attend_one", "kind": "attend", "batch": 1, "lo": 300, "hi": 300, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "width": 32, "type": "bf16", "kv": "bf16",
         "lse": False, "mix": 1},
        # a small server's step: 16 requests between the benchmark's first and last position
        {"name": "attend_step", "kind": "attend", "batch": 16, "lo": 257, "hi": 1280, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "width": 128, "type": "bf16", "kv": "bf16",
         "lse": False, "mix": 2},
        # a full server: 128 requests from just begun to 8000 positions, one slot empty
        {"name": "attend_ragged", "kind": "attend", "batch": 128, "lo": 0, "hi": 8000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "width": 256, "type": "bf16", "kv": "bf16",
         "lse": False, "mix": 3},
        # one very long document; the log-sum-exp is kept to join other parts
        {"name": "attend_long", "kind": "attend", "batch": 1, "lo": 131001, "hi": 131001,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "width": 2048, "type": "bf16",
         "kv": "bf16", "lse": True, "mix": 4},
        # the same server with an 8-bit cache
        {"name": "attend_e4m3", "kind": "attend", "batch": 64, "lo": 500, "hi": 6000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "width": 192, "type": "bf16", "kv": "e4m3",
         "lse": False, "mix": 5},
        # float16, short heads, many query heads over two key heads
        {"name": "attend_f16_64", "kind": "attend", "batch": 24, "lo": 1, "hi": 3500, "heads": 40,
         "kv_heads": 2, "dim": 64, "page": 16, "width": 220, "type": "f16", "kv": "f16",
         "lse": True, "mix": 6},
        # a step's 16 rows into their caches
        {"name": "write_step", "kind": "write", "seqs": 16, "rows_each": 1, "past": 1280,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "kv": "bf16",
         "norm": True, "pad": 0, "mix": 7},
        # three prompts of 1100 rows (text and a reference clip) into an 8-bit cache
        {"name": "write_prompt_e4m3", "kind": "write", "seqs": 3, "rows_each": 1100, "past": 0,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "type": "bf16", "kv": "e4m3",
         "norm": True, "pad": 64, "mix": 8},
        # two candidates of one sentence, eight layers
        {"name": "branch_two", "kind": "branch", "layers": 8, "pages": 256, "page": 16,
         "kv_heads": 8, "dim": 128, "parents": 1, "each": 2, "lo": 700, "hi": 700, "add": 1,
         "width": 64, "type": "bf16", "mix": 9},
        # 16 sentences with four candidates each, all 36 layers of the backbone
        {"name": "branch_server", "kind": "branch", "layers": 36, "pages": 700, "page": 16,
         "kv_heads": 8, "dim": 128, "parents": 16, "each": 4, "lo": 60, "hi": 500, "add": 20,
         "width": 128, "type": "bf16", "mix": 10},
        # a small pool after a few requests have ended
        {"name": "compact_small", "kind": "compact", "layers": 8, "pages": 300, "page": 16,
         "kv_heads": 8, "dim": 128, "seqs": 12, "live": 0.4, "shared": 2, "width": 40,
         "type": "bf16", "mix": 11},
        # a server's pool, half empty, 36 layers
        {"name": "compact_server", "kind": "compact", "layers": 36, "pages": 900, "page": 32,
         "kv_heads": 8, "dim": 128, "seqs": 40, "live": 0.5, "shared": 8, "width": 64,
         "type": "bf16", "mix": 12},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(("attend", "attend", "attend", "write", "write", "branch", "compact"))
    mix = rng.randrange(1 << 30)
    kv_heads, group = rng.choice(((8, 4), (8, 4), (8, 2), (4, 7), (8, 1), (2, 20), (1, 8), (8, 8)))
    dim = rng.choice((128, 128, 128, 64))
    page = rng.choice((16, 16, 32, 64, 128))
    kind16 = rng.choice(("bf16", "bf16", "f16"))
    kv = rng.choice((kind16, kind16, "e4m3"))

    def layers(pages):                                        # a pool of at most 4 GB
        return max(1, min(rng.randint(1, 16), 4 * 10**9 // (pages * page * kv_heads * dim * 4)))

    if kind == "attend":
        batch = _log(rng, 1, 128)
        # no more than about 400000 positions of 8 heads of 128 (the largest listed case)
        most = max(8, min(131072, 400_000 // batch * 1024 // (kv_heads * dim)))
        hi = _log(rng, 1, most)
        lo = rng.choice((0, 1, hi // 2, hi))
        return {"kind": kind, "batch": batch, "lo": min(lo, hi), "hi": hi,
                "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page,
                "width": -(-hi // page) + rng.randint(0, 9), "type": kind16, "kv": kv,
                "lse": rng.random() < 0.3, "mix": mix}
    if kind == "write":
        seqs = _log(rng, 1, 64)
        return {"kind": kind, "seqs": seqs, "rows_each": _log(rng, 1, max(1, 4000 // seqs)),
                "past": _log(rng, 1, 4000) - 1, "heads": kv_heads * group, "kv_heads": kv_heads,
                "dim": dim, "page": page, "type": kind16, "kv": kv, "norm": rng.random() < 0.7,
                "pad": rng.choice((0, 0, 8, 128)), "mix": mix}
    if kind == "branch":
        parents, each, add = _log(rng, 1, 20), rng.randint(1, 4), _log(rng, 1, 60)
        hi = _log(rng, 3, 500)
        need = parents * -(-hi // page) + parents * each * (2 + -(-add // page))
        pages = need + rng.randint(0, 40)
        return {"kind": kind, "layers": layers(pages), "pages": pages,
                "page": page, "kv_heads": kv_heads, "dim": dim, "parents": parents, "each": each,
                "lo": 1, "hi": hi, "add": add, "width": -(-(hi + add) // page) + rng.randint(0, 5),
                "type": kind16, "mix": mix}
    pages = _log(rng, 40, 900)
    return {"kind": kind, "layers": layers(pages), "pages": pages, "page": page,
            "kv_heads": kv_heads, "dim": dim, "seqs": rng.randint(2, 30),
            "live": round(rng.uniform(0.1, 0.9), 3), "shared": rng.randint(0, 8), "width": 70,
            "type": kind16, "mix": mix}


# ------------------------------------------------------------------------------ inputs
def _lens(case) -> list[int]:
    """The sequences' lengths, spread over their logarithm; a batch that may hold an empty slot
    holds one."""
    rng = random.Random(case["mix"])
    lo, hi = case["lo"], case["hi"]
    n = case["batch"] if case["kind"] == "attend" else case["parents"]
    lens = [_log(rng, max(lo, 1), hi) if hi > 0 else 0 for _ in range(n)]
    lens[rng.randrange(n)] = hi
    if lo == 0 and n > 1:
        lens[0 if lens[0] != hi else 1] = 0
    return lens


def _gen(seed: int, stream: int = 0) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1009 + stream)
    return g


def _pool(gen, kv: str, *shape) -> torch.Tensor:
    """A page pool of normal values, filled a layer (or a block of pages) at a time."""
    out = torch.empty(*shape, dtype=_TYPES[kv], device="cuda")
    step = max(1, (1 << 26) // max(1, out[0].numel()))
    for i in range(0, shape[0], step):
        block = torch.randn(out[i:i + step].shape, device="cuda", generator=gen)
        out[i:i + step] = block.to(_TYPES[kv])
    return out


def _table(gen, lens: list[int], page: int, width: int, rows: int, pages: int) -> torch.Tensor:
    """Pages in a shuffled order: row i has those of lens[i], -1 behind them."""
    need = torch.tensor([-(-n // page) for n in lens] + [0] * (rows - len(lens)), device="cuda")
    first = need.cumsum(0) - need
    order = torch.randperm(pages, device="cuda", generator=gen)
    j = torch.arange(width, device="cuda")[None]
    at = (first[:, None] + j).clamp(max=pages - 1)
    return torch.where(j < need[:, None], order[at], -1).int().contiguous()


def _scales(gen, case):
    if case["kv"] != "e4m3":
        return None, None
    h = case["kv_heads"]
    return (torch.rand(h, device="cuda", generator=gen) * 0.5 + 0.75,
            torch.rand(h, device="cuda", generator=gen) * 0.5 + 0.75)


def prepare(case, seed) -> dict:
    gen = _gen(seed)
    kind, page, dim, hkv = case["kind"], case["page"], case["dim"], case["kv_heads"]
    st = {"kind": kind, "page": page}
    if kind == "attend":
        lens = _lens(case)
        pages = max(1, sum(-(-n // page) for n in lens)) + 3
        st["k"] = _pool(gen, case["kv"], pages, hkv, page, dim)
        st["v"] = _pool(gen, case["kv"], pages, hkv, page, dim)
        st["q"] = torch.randn(case["batch"], case["heads"], dim, device="cuda",
                              generator=gen).to(_TYPES[case["type"]])
        st["table"] = _table(gen, lens, page, case["width"], len(lens), pages)
        st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["k_scale"], st["v_scale"] = _scales(gen, case)
        st["scale"], st["lse"] = dim ** -0.5, case["lse"]
    elif kind == "write":
        n, each, past = case["seqs"], case["rows_each"], case["past"]
        width = -(-(past + each) // page) + 1
        need = -(-(past + each) // page) - past // page     # only pages that take new rows exist
        pages = n * need + 2
        st["k"] = _pool(gen, case["kv"], pages, hkv, page, dim)
        st["v"] = _pool(gen, case["kv"], pages, hkv, page, dim)
        cols = (case["heads"] + 2 * hkv) * dim
        rows = n * each
        buf = torch.randn(rows, cols + case["pad"], device="cuda", generator=gen)
        st["qkv"] = buf.to(_TYPES[case["type"]])[:, :cols]
        j = torch.arange(width, device="cuda")
        order = torch.randperm(pages, device="cuda", generator=gen)
        slot = torch.arange(n, device="cuda")[:, None] * need + (j - past // page)[None]
        has = (j >= past // page) & (j < past // page + need)
        st["table"] = torch.where(has[None], order[slot.clamp(0, pages - 1)], -1).int().contiguous()
        st["positions"] = (past + torch.arange(each, device="cuda")).repeat(n)
        st["seqs"] = torch.arange(n, device="cuda").repeat_interleave(each).int()
        st["q_norm"] = st["k_norm"] = st["cos"] = st["sin"] = None
        if case["norm"]:
            st["q_norm"], st["k_norm"] = (
                (1 + 0.05 * torch.randn(dim, device="cuda", generator=gen)).to(_TYPES[case["type"]])
                for _ in range(2))
            inv = THETA ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
            ang = torch.outer(torch.arange(width * page, device="cuda", dtype=torch.float64), inv)
            st["cos"] = torch.cat([ang.cos()] * 2, -1).float()
            st["sin"] = torch.cat([ang.sin()] * 2, -1).float()
        st["k_scale"], st["v_scale"] = _scales(gen, case)
        st["heads"] = case["heads"]
    elif kind == "branch":
        lens = _lens(case)
        n, each, pages = case["parents"], case["each"], case["pages"]
        st["k"] = _pool(gen, case["type"], case["layers"], pages, hkv, page, dim)
        st["v"] = _pool(gen, case["type"], case["layers"], pages, hkv, page, dim)
        st["table"] = _table(gen, lens, page, case["width"], n * (1 + each), pages)
        st["lens"] = torch.tensor(lens + [0] * (n * each), dtype=torch.int32, device="cuda")
        st["refs"] = _counts(st["table"], pages)
        st["parents"] = torch.arange(n, device="cuda").repeat_interleave(each).int()
        st["children"] = (n + torch.arange(n * each, device="cuda")).int()
        st["zeros"] = torch.zeros(n * each, dtype=torch.int32, device="cuda")
        st["counts"] = torch.full((n * each,), case["add"], dtype=torch.int32, device="cuda")
    else:
        lens, shared = _fragments(case)
        pages = case["pages"]
        st["k"] = _pool(gen, case["type"], case["layers"], pages, hkv, page, dim)
        st["v"] = _pool(gen, case["type"], case["layers"], pages, hkv, page, dim)
        st["table"] = _table(gen, lens, page, case["width"], case["seqs"] + len(shared), pages)
        for i, s in enumerate(shared):                       # forks: rows that share all pages
            st["table"][case["seqs"] + i] = st["table"][s]
        st["refs"] = _counts(st["table"], pages)
    return st


def _counts(table, pages: int) -> torch.Tensor:
    flat = table.reshape(-1).long()
    return torch.zeros(pages + 1, dtype=torch.int32, device="cuda").index_add_(
        0, torch.where(flat < 0, pages, flat),
        torch.ones_like(flat, dtype=torch.int32))[:pages].contiguous()


def _fragments(case):
    """Lengths whose pages fill the live share of the pool, and the sequences that are shared."""
    rng = random.Random(case["mix"])
    left, lens = max(1, int(case["pages"] * case["live"])), []
    for i in range(case["seqs"]):
        want = min(case["width"], max(0, left // (case["seqs"] - i)))
        lens.append(want * case["page"])
        left -= want
    return lens, [rng.randrange(case["seqs"]) for _ in range(case["shared"])]


# ------------------------------------------------------------------------------ one pass
_paged = None


def _framework():
    global _paged
    if _paged is None:
        import __graft_entry__

        __graft_entry__.import_package()
        from moss_tts_lite_amd import paged

        _paged = paged
    return _paged


def run(st):
    if st["kind"] == "attend":
        return _run_own_attend(st) if own else _attend(st)
    if st["kind"] == "write":
        return _run_own_write(st) if own else _write(st)
    if st["kind"] == "branch":
        return _run_own_branch(st) if own else _branch(st)
    return _run_own_compact(st) if own else _compact(st)


def _run_own_attend(st):
    p = _framework()
    if st["lse"]:
        out, lse = p.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"],
                                     st["scale"], st["k_scale"], st["v_scale"], return_lse=True)
        return {"out": out, "lse": lse}
    return {"out": p.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"],
                                     st["scale"], st["k_scale"], st["v_scale"])}


def _run_own_write(st):
    q = _framework().paged_write(st["qkv"], st["k"], st["v"], st["table"], st["positions"],
                                 st["seqs"], st["q_norm"], st["k_norm"], st["cos"], st["sin"], EPS,
                                 st["k_scale"], st["v_scale"])
    return {"q": q, "k": st["k"], "v": st["v"]}


def _run_own_branch(st):
    p = _framework()
    a = (st["table"], st["lens"], st["refs"])
    s0 = p.pages_truncate(*a, st["children"], st["zeros"], st["page"])
    s1 = p.pages_fork(*a, st["parents"], st["children"], st["page"])
    s2 = p.pages_extend(*a, st["children"], st["counts"], st["k"], st["v"])
    return {"table": a[0], "lens": a[1], "refs": a[2], "k": st["k"], "v": st["v"],
            "status": [s0, s1, s2]}


def _run_own_compact(st):
    table, refs, live = _framework().pages_compact(st["table"], st["refs"], st["k"], st["v"])
    return {"table": table, "refs": refs, "live": live, "k": st["k"], "v": st["v"]}


# ------------------------------------------------------------------------------ plain forms
def _attend(st):
    q, table, lens = st["q"], st["table"].long(), st["lens"]
    b, heads, dim = q.shape
    hkv = st["k"].shape[1]

    def rows(pages, scale):
        x = pages[table.clamp(min=0)].float()                # [b, width, hkv, page, dim]
        if scale is not None:
            x = x * scale[:, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, dim)

    k, v = rows(st["k"], st["k_scale"]), rows(st["v"], st["v_scale"])
    s = torch.matmul(q.float().reshape(b, hkv, -1, dim), k.transpose(-1, -2)) * st["scale"]
    n = k.shape[2]
    keep = torch.arange(n, device=q.device)[None] < lens[:, None]
    keep = (keep & (table >= 0).repeat_interleave(st["page"], 1))[:, None, None]
    s = s.masked_fill(~keep, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.reshape(b, heads, dim).to(q.dtype)
    if st["lse"]:
        return {"out": out, "lse": (top + torch.log(total)).reshape(b, heads)}
    return {"out": out}


def _norm_rope(x, w, st):
    if w is None:
        return x
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    half = x.shape[-1] // 2
    c, s = (t[st["positions"]][:, None] for t in (st["cos"], st["sin"]))
    return x * c + torch.cat([-x[..., half:], x[..., :half]], -1) * s


def _store(x, pages, scale):
    if pages.dtype == torch.float8_e4m3fn:
        x = (x / scale[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
    return x.to(pages.dtype)


def _write(st):
    qkv, heads = st["qkv"], st["heads"]
    rows, dim, hkv = qkv.shape[0], st["k"].shape[3], st["k"].shape[1]
    x = qkv.float().reshape(rows, -1, dim)
    q = _norm_rope(x[:, :heads], st["q_norm"], st).to(qkv.dtype)
    k = _norm_rope(x[:, heads:heads + hkv], st["k_norm"], st)
    at = st["table"][st["seqs"].long(), st["positions"] // st["page"]].long()
    off = st["positions"] % st["page"]
    u8 = torch.uint8 if st["k"].dtype == torch.float8_e4m3fn else st["k"].dtype
    st["k"].view(u8)[at, :, off] = _store(k, st["k"], st["k_scale"]).view(u8)
    st["v"].view(u8)[at, :, off] = _store(x[:, heads + hkv:], st["v"], st["v_scale"]).view(u8)
    return {"q": q, "k": st["k"], "v": st["v"]}


def _truncate(st, seqs, new):
    table, lens, refs = st["table"], st["lens"], st["refs"]
    seqs = seqs.long()
    rows = table[seqs]
    ok = ((new >= 0) & (new <= lens[seqs])).all()
    j = torch.arange(table.shape[1], device=table.device)[None]
    drop = (j >= ((new + st["page"] - 1) // st["page"])[:, None]) & (rows >= 0) & ok
    refs.index_add_(0, rows.clamp(min=0).reshape(-1).long(), -drop.reshape(-1).int())
    table[seqs] = torch.where(drop, -1, rows)
    lens[seqs] = torch.where(ok, new, lens[seqs])
    return torch.where(ok, 0, 2).int().reshape(1)


def _fork(st, parents, children):
    table, lens, refs = st["table"], st["lens"], st["refs"]
    parents, children = parents.long(), children.long()
    rows = table[parents]
    ok = (lens[children] == 0).all()
    refs.index_add_(0, rows.clamp(min=0).reshape(-1).long(), ((rows >= 0) & ok).reshape(-1).int())
    table[children] = torch.where(ok, rows, table[children])
    lens[children] = torch.where(ok, lens[parents], lens[children])
    return torch.where(ok, 0, 2).int().reshape(1)


def _extend(st, seqs, counts):
    table, lens, refs, page = st["table"], st["lens"], st["refs"], st["page"]
    seqs = seqs.long()
    rows, have = table[seqs].long(), lens[seqs].long()
    n, width = rows.shape
    j = torch.arange(width, device=rows.device)[None]
    used, want = -(-have // page), -(-(have + counts) // page)
    # a partly filled last page that others hold too: copied, but for the last holder of a call
    last = rows.gather(1, (have // page).clamp(max=width - 1)[:, None])[:, 0].clamp(min=0)
    part = (have % page > 0) & (counts > 0)
    earlier = (last[:, None] == last[None]) & part[:, None] & part[None]
    rank = torch.tril(earlier, -1).sum(1)
    cow = part & (refs[last] - rank > 1)
    fresh = ((j >= used[:, None]) & (j < want[:, None])) | (cow[:, None] & (j == (have // page)[:, None]))
    order = (fresh.reshape(-1).cumsum(0) - 1).reshape(n, width)
    free = torch.argsort((refs != 0).int(), stable=True)      # free pages first, lowest first
    enough = fresh.sum() <= (refs == 0).sum()
    ok = enough & (want <= width).all() & (counts >= 0).all()
    page_of = free[order.clamp(0, refs.numel() - 1)]
    fresh, cow = fresh & ok, cow & ok
    dst = page_of.gather(1, (have // page).clamp(max=width - 1)[:, None])[:, 0]
    first = torch.argmax(cow.int())                           # nothing to copy: the first copy again,
    src = torch.where(cow, last, last[first])                 # or, where there is none, onto itself
    dst = torch.where(cow, dst, torch.where(cow[first], dst[first], last[first]))
    refs.index_add_(0, last, -cow.int())
    refs.index_add_(0, page_of.reshape(-1), fresh.reshape(-1).int())
    table[seqs] = torch.where(fresh, page_of, rows).int()
    lens[seqs] = torch.where(ok, have + counts, have).int()
    for x in (st["k"], st["v"]):
        x[:, dst] = x[:, src]
    return torch.where(ok, 0, torch.where(enough, 2, 1)).int().reshape(1)


def _branch(st):
    s0 = _truncate(st, st["children"], st["zeros"])
    s1 = _fork(st, st["parents"], st["children"])
    s2 = _extend(st, st["children"], st["counts"])
    return {"table": st["table"], "lens": st["lens"], "refs": st["refs"], "k": st["k"],
            "v": st["v"], "status": [s0, s1, s2]}


def _compact(st):
    table, refs = st["table"], st["refs"]
    pages = refs.numel()
    at = torch.arange(pages, device=refs.device)
    alive = refs > 0
    live = alive.sum()
    mover, hole = alive & (at >= live), ~alive & (at < live)
    movers = torch.argsort((~mover).int(), stable=True)[:pages // 2]
    holes = torch.argsort((~hole).int(), stable=True)[:pages // 2]
    moves = at[:pages // 2] < mover.sum()
    src = torch.where(moves, movers, pages - 1)               # the last page onto itself
    dst = torch.where(moves, holes, pages - 1)
    goes = at.clone()
    goes[src] = dst
    goes[pages - 1] = torch.where(mover[pages - 1], holes[(mover.sum() - 1).clamp(0)], pages - 1)
    new_refs = torch.zeros_like(refs).index_add_(0, goes, torch.where(alive, refs, 0))
    new_table = torch.where(table >= 0, goes[table.clamp(min=0).long()].int(), table)
    for x in (st["k"], st["v"]):
        x[:, dst] = x[:, src]
    return {"table": new_table, "refs": new_refs, "live": live.int().reshape(1), "k": st["k"],
            "v": st["v"]}


# ------------------------------------------------------------------------------ work
def work(case) -> dict:
    kind, page, dim, hkv = case["kind"], case["page"], case["dim"], case["kv_heads"]
    size = 1 if case.get("kv") == "e4m3" else 2
    if kind == "attend":
        total, b, heads = sum(_lens(case)), case["batch"], case["heads"]
        return {"bytes": 2 * total * hkv * dim * size + 4 * b * heads * dim + 4 * (total // page + b)
                + (4 * b * heads if case["lse"] else 0),
                "flops": 4 * total * heads * dim}
    if kind == "write":
        rows = case["seqs"] * case["rows_each"]
        tables = 8 * case["rows_each"] * dim if case["norm"] else 0
        return {"bytes": rows * dim * (2 * (2 * case["heads"] + 2 * hkv) + 2 * hkv * size) + tables
                + 12 * rows,
                "flops": 10 * rows * (case["heads"] + 2 * hkv) * dim}
    one = 2 * case["layers"] * hkv * page * dim * 2           # a page of all layers, K and V
    if kind == "branch":
        lens, n = _lens(case), case["parents"] * case["each"]
        copies = sum(case["each"] for x in lens if x % page)
        held = sum(-(-x // page) for x in lens) * case["each"]
        return {"bytes": 2 * copies * one + 4 * (6 * held + 8 * n) + 4 * case["pages"], "flops": 0}
    # the pages above the live count are a random share of the pool
    lens, _ = _fragments(case)
    live = sum(x // page for x in lens)
    moves = live * (case["pages"] - live) // case["pages"]
    return {"bytes": 2 * moves * one + 8 * case["pages"]
            + 8 * (case["seqs"] + case["shared"]) * case["width"], "flops": 0}


# ------------------------------------------------------------------------------ definitions
def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "attend":
        return _exact_attend(st)
    if st["kind"] == "write":
        return _exact_write(st)
    return _exact_branch(st) if st["kind"] == "branch" else _exact_compact(st)


def _exact_attend(st):
    """Sequence by sequence over exactly its positions, in float64."""
    q, page = st["q"].double(), st["page"]
    b, heads, dim = q.shape
    hkv = st["k"].shape[1]
    out = torch.zeros(b, heads, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((b, heads), float("-inf"), dtype=torch.float64, device=q.device)
    for i, n in enumerate(st["lens"].tolist()):
        if n == 0:
            continue
        ids = st["table"][i, :-(-n // page)].long()
        for h in range(hkv):
            k, v = (x[ids, h].reshape(-1, dim)[:n].double() for x in (st["k"], st["v"]))
            if st["k_scale"] is not None:
                k, v = k * float(st["k_scale"][h]), v * float(st["v_scale"][h])
            g = slice(h * (heads // hkv), (h + 1) * (heads // hkv))
            s = (k @ q[i, g].T).T * st["scale"]
            lse[i, g] = torch.logsumexp(s, -1)
            out[i, g] = torch.softmax(s, -1) @ v
    return {"out": out, "lse": lse} if st["lse"] else {"out": out}


def _exact_write(st):
    qkv = st["qkv"].double()
    heads, hkv, page, dim = st["heads"], st["k"].shape[1], st["page"], st["k"].shape[3]
    x = qkv.reshape(qkv.shape[0], -1, dim).clone()
    if st["q_norm"] is not None:
        half = dim // 2
        for h in range(heads + hkv):
            w = (st["q_norm"] if h < heads else st["k_norm"]).double()
            y = x[:, h] / (x[:, h].square().sum(-1, keepdim=True) / dim + EPS).sqrt() * w
            c = st["cos"].double()[st["positions"]]
            s = st["sin"].double()[st["positions"]]
            x[:, h, :half] = y[:, :half] * c[:, :half] - y[:, half:] * s[:, :half]
            x[:, h, half:] = y[:, half:] * c[:, half:] + y[:, :half] * s[:, half:]
    k, v = st["k"].double(), st["v"].double()
    table, seqs = st["table"].tolist(), st["seqs"].tolist()
    for i, pos in enumerate(st["positions"].tolist()):
        pid = table[seqs[i]][pos // page]
        for dst, part, scale in ((k, x[i, heads:heads + hkv], st["k_scale"]),
                                 (v, x[i, heads + hkv:], st["v_scale"])):
            if scale is not None:
                part = (part / scale.double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
            dst[pid, :, pos % page] = part
    return {"q": x[:, :heads], "k": k, "v": v}


def _exact_branch(st):
    """The three calls, one entry after the other on the host."""
    page = st["page"]
    table, lens, refs = st["table"].tolist(), st["lens"].tolist(), st["refs"].tolist()
    width, copies = len(table[0]), []
    for s in st["children"].tolist():                         # dropped
        for j in range(width):
            if table[s][j] >= 0:
                refs[table[s][j]] -= 1
                table[s][j] = -1
        lens[s] = 0
    for p, c in zip(st["parents"].tolist(), st["children"].tolist()):
        table[c], lens[c] = list(table[p]), lens[p]
        for x in table[c]:
            if x >= 0:
                refs[x] += 1
    for s, n in zip(st["children"].tolist(), st["counts"].tolist()):
        at = lens[s] // page
        if n > 0 and lens[s] % page and refs[table[s][at]] > 1:
            new = refs.index(0)
            copies.append((table[s][at], new))
            refs[table[s][at]] -= 1
            refs[new], table[s][at] = 1, new
        for j in range(-(-lens[s] // page), -(-(lens[s] + n) // page)):
            new = refs.index(0)
            refs[new], table[s][j] = 1, new
        lens[s] += n
    k, v = st["k"].clone(), st["v"].clone()
    for a, b in copies:
        k[:, b], v[:, b] = k[:, a], v[:, a]
    return {"table": torch.tensor(table), "lens": torch.tensor(lens), "refs": torch.tensor(refs),
            "k": k, "v": v, "status": [torch.zeros(1, dtype=torch.int32)] * 3}


def _exact_compact(st):
    table, refs = st["table"].tolist(), st["refs"].tolist()
    live = sum(r > 0 for r in refs)
    k, v = st["k"].clone(), st["v"].clone()
    goes = {}
    for p in range(live, len(refs)):
        if refs[p] > 0:
            new = refs.index(0)
            goes[p] = new
            refs[new], refs[p] = refs[p], 0
            k[:, new], v[:, new] = k[:, p], v[:, p]
    table = [[goes.get(x, x) for x in row] for row in table]
    return {"table": torch.tensor(table), "refs": torch.tensor(refs),
            "live": torch.tensor([live]), "k": k, "v": v}
