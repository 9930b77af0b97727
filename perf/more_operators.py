"""What is timed of a step of several sequences around the paged key-value cache: norms and
rotation of queries and keys, attention of sequences that share a prefix, and the draw of the next
tokens.

``listed()`` names the cases, ``draw(rng)`` gives others of the same ranges, ``prepare`` builds
what a program holds before the call, ``run`` is one pass: with ``own`` through the framework's
entry points, else in plain torch operations.  ``exact`` computes the same from the definitions in
float64, ``work`` is what a pass cannot do without.

Three kinds of case:

* ``shared``: one query token of each sequence over its pages, where consecutive sequences form
  groups whose first positions lie in the same pages (candidates of a sentence, requests on one
  voice prompt);
* ``sample``: the next token of each row of logits by temperature, top-k, top-p and min-p from
  given random numbers, and the logarithm of its probability;
* ``rotary``: RMSNorm of each head of q and k and the rotation by position, out of a q | k | v
  matrix.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

THETA, EPS = 1_000_000.0, 1e-6
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn,
          "f32": torch.float32}


def listed() -> list[dict]:
    return [
        # the smallest call: two candidates of one sentence, just forked behind its prompt
        {"name": "shared_two", "kind": "shared", "groups": 1, "each_lo": 2, "each": 2,
         "shared_lo": 700, "shared": 700, "own_lo": 1, "own": 30, "empty": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "room": 20, "type": "bf16", "kv": "bf16",
         "lse": False, "mix": 1},
        # 16 sentences with up to six candidates each, between their prompts' ends and 600 steps on
        {"name": "shared_candidates", "kind": "shared", "groups": 16, "each_lo": 2, "each": 6,
         "shared_lo": 257, "shared": 1100, "own_lo": 1, "own": 600, "empty": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "room": 10, "type": "bf16", "kv": "bf16",
         "lse": False, "mix": 2},
        # a full server whose 192 requests speak with one voice: a long reference prompt
        {"name": "shared_voice", "kind": "shared", "groups": 1, "each_lo": 192, "each": 192,
         "shared_lo": 6001, "shared": 6001, "own_lo": 1, "own": 700, "empty": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "room": 3, "type": "bf16", "kv": "bf16",
         "lse": False, "mix": 3},
        # five voices of 1 to 24 requests each in an 8-bit cache; the log-sum-exp is kept
        {"name": "shared_e4m3", "kind": "shared", "groups": 5, "each_lo": 1, "each": 24,
         "shared_lo": 1500, "shared": 8000, "own_lo": 1, "own": 1000, "empty": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "room": 0, "type": "bf16", "kv": "e4m3",
         "lse": True, "mix": 4},
        # float16, short heads, 20 query heads to each of two key heads, pages that end inside
        {"name": "shared_f16_64", "kind": "shared", "groups": 3, "each_lo": 3, "each": 17,
         "shared_lo": 999, "shared": 3500, "own_lo": 1, "own": 300, "empty": True, "heads": 40,
         "kv_heads": 2, "dim": 64, "page": 64, "room": 5, "type": "f16", "kv": "f16",
         "lse": True, "mix": 5},
        # one text token out of the full vocabulary, as a sentence's generation draws it
        {"name": "sample_text", "kind": "sample", "rows": 1, "vocab": 151936, "type": "bf16",
         "how": "all", "temperature": 1.5, "top_k": 50, "top_p": 1.0, "min_p": 0.0, "mix": 6},
        # one frame's 31 audio channels
        {"name": "sample_audio", "kind": "sample", "rows": 31, "vocab": 1025, "type": "bf16",
         "how": "all", "temperature": 1.7, "top_k": 25, "top_p": 0.8, "min_p": 0.0, "mix": 7},
        # a server's step: 96 requests, each with settings of its own (greedy ones among them)
        {"name": "sample_server", "kind": "sample", "rows": 96, "vocab": 151936, "type": "f32",
         "how": "rows", "temperature": 1.0, "top_k": 50, "top_p": 0.9, "min_p": 0.05, "mix": 8},
        # 24 candidates by top-p alone: how many tokens that keeps is not known beforehand
        {"name": "sample_nucleus", "kind": "sample", "rows": 24, "vocab": 151936, "type": "bf16",
         "how": "all", "temperature": 0.9, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "mix": 9},
        # a step's 16 rows, two pad rows behind them
        {"name": "rotary_step", "kind": "rotary", "rows": 18, "pads": 2, "heads": 32,
         "kv_heads": 8, "dim": 128, "turned": 128, "interleaved": False, "amplitude": 1.0,
         "norm": True, "far": 1280, "pad": 0, "type": "bf16", "mix": 10},
        # three prompts of 1100 rows, half of each head turned, neighbouring dims as pairs, no norm
        {"name": "rotary_prompt", "kind": "rotary", "rows": 3300, "pads": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "turned": 64, "interleaved": True, "amplitude": 1.0,
         "norm": False, "far": 4000, "pad": 64, "type": "f16", "mix": 11},
        # 16000 rows of long documents near position 10^6, frequencies and amplitude scaled
        {"name": "rotary_far", "kind": "rotary", "rows": 16000, "pads": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "turned": 128, "interleaved": False, "amplitude": 1.2,
         "norm": True, "far": 1_000_000, "pad": 0, "type": "bf16", "mix": 12},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(("shared", "shared", "shared", "sample", "sample", "rotary"))
    mix = rng.randrange(1 << 30)
    kind16 = rng.choice(("bf16", "bf16", "f16"))
    kv_heads, group = rng.choice(((8, 4), (8, 4), (8, 2), (4, 7), (8, 1), (2, 20), (1, 8), (8, 8)))
    dim = rng.choice((128, 128, 128, 64))
    if kind == "shared":
        batch = _log(rng, 2, 192)
        groups = _log(rng, 1, batch)
        each = -(-batch // groups)
        # no more than a million positions of 32 heads of 128 over 8, all sequences by themselves
        most = max(8, min(40000, 1_000_000 // (groups * each) * 1024 // (kv_heads * dim),
                          1_000_000 // (groups * each) * 4096 // (kv_heads * group * dim)))
        shared = _log(rng, 1, most)
        return {"kind": kind, "groups": groups, "each_lo": rng.choice((1, each)), "each": each,
                "shared_lo": rng.choice((0, shared // 2, shared)), "shared": shared,
                "own_lo": rng.choice((0, 1)), "own": _log(rng, 1, max(1, min(2000, most // 8))),
                "empty": rng.random() < 0.3, "heads": kv_heads * group, "kv_heads": kv_heads,
                "dim": dim, "page": rng.choice((16, 16, 32, 64, 128, 256)),
                "room": rng.randint(0, 9), "type": kind16, "kv": rng.choice((kind16, "e4m3")),
                "lse": rng.random() < 0.4, "mix": mix}
    if kind == "sample":
        vocab = _log(rng, 2, 152000)
        return {"kind": kind, "rows": _log(rng, 1, min(512, 12_000_000 // vocab)), "vocab": vocab,
                "type": rng.choice(("bf16", "f16", "f32")), "how": rng.choice(("all", "rows")),
                "temperature": round(rng.uniform(0.4, 1.8), 3),
                "top_k": rng.choice((0, 0, 1, _log(rng, 1, 2000))),
                "top_p": rng.choice((1.0, round(rng.uniform(0.05, 0.99), 3))),
                "min_p": rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.3), 4))), "mix": mix}
    heads, wide = kv_heads * group, rng.choice((64, 80, 96, 128, 128, 192, 256))
    interleaved = rng.random() < 0.4
    return {"kind": kind, "rows": _log(rng, 1, 16000 * 40 * 128 // ((heads + kv_heads) * wide)),
            "pads": rng.choice((0, 0, 1, 3)), "heads": heads, "kv_heads": kv_heads, "dim": wide,
            "turned": rng.choice((wide, wide, wide // 2, 16)), "interleaved": interleaved,
            "amplitude": rng.choice((1.0, round(rng.uniform(0.8, 1.5), 3))),
            "norm": rng.random() < 0.7, "far": _log(rng, 1, 2_000_000), "pad": rng.choice((0, 8, 128)),
            "type": kind16, "mix": mix}


# ------------------------------------------------------------------------------ inputs
def _layout(case):
    """(sequences of each group, shared positions of each group, length of each sequence)"""
    rng = random.Random(case["mix"])
    sizes = [rng.randint(case["each_lo"], case["each"]) for _ in range(case["groups"])]
    sizes[rng.randrange(len(sizes))] = case["each"]
    shared, lens = [], []
    for n in sizes:
        lo = case["shared_lo"]
        s = 0 if lo == 0 and rng.random() < 0.3 else _log(rng, max(1, lo), case["shared"])
        shared.append(s)
        for _ in range(n):
            none = case["own_lo"] == 0 and rng.random() < 0.2
            lens.append(s if none else s + _log(rng, 1, case["own"]))
    if case["empty"] and len(lens) > 1:                      # a finished candidate's slot
        lens[rng.randrange(1, len(lens))] = 0
    return sizes, shared, lens


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1009)
    return g


def _pool(gen, kv: str, *shape) -> torch.Tensor:
    out = torch.empty(*shape, dtype=_TYPES[kv], device="cuda")
    step = max(1, (1 << 26) // max(1, out[0].numel()))
    for i in range(0, shape[0], step):
        block = torch.randn(out[i:i + step].shape, device="cuda", generator=gen)
        out[i:i + step] = block.to(_TYPES[kv])
    return out


def prepare(case, seed) -> dict:
    gen = _gen(seed)
    st = {"kind": case["kind"]}
    if case["kind"] == "shared":
        _prepare_shared(case, gen, st)
    elif case["kind"] == "sample":
        _prepare_sample(case, gen, st)
    else:
        _prepare_rotary(case, gen, st)
    return st


def _prepare_shared(case, gen, st) -> None:
    page, dim, hkv = case["page"], case["dim"], case["kv_heads"]
    sizes, shared, lens = _layout(case)
    width = max(1, max(-(-n // page) for n in lens)) + case["room"]
    # whole shared pages are held by all of a group; a partly shared page has been copied when its
    # holders were extended, so its shared rows are alike in all of them
    rows, same, at, nxt = [], [], 0, 0
    for n, s in zip(sizes, shared):
        trunk = list(range(nxt, nxt + s // page))
        nxt += len(trunk)
        first = None
        for i in range(n):
            have = -(-lens[at] // page)
            mine = list(range(nxt, nxt + max(0, have - len(trunk))))
            nxt += len(mine)
            if s % page and mine:
                if first is None:
                    first = mine[0]
                same.append((mine[0], first, s % page))
            rows.append((trunk if have else []) + mine)
            at += 1
    pages = nxt + 3
    k, v = (_pool(gen, case["kv"], pages, hkv, page, dim) for _ in range(2))
    u8 = torch.uint8 if case["kv"] == "e4m3" else k.dtype
    if same:
        to, of, n = torch.tensor(same, device="cuda").T
        alike = (torch.arange(page, device="cuda")[None] < n[:, None])[:, None, :, None]
        for x in (k.view(u8), v.view(u8)):
            x[to] = torch.where(alike, x[of], x[to])
    order = torch.randperm(pages, device="cuda", generator=gen)
    back = torch.empty_like(order)
    back[order] = torch.arange(pages, device="cuda")
    st["k"], st["v"] = (x.view(u8)[back].view(x.dtype) for x in (k, v))
    flat = torch.full((len(lens), width), -1, dtype=torch.int64)
    for i, r in enumerate(rows):
        flat[i, :len(r)] = torch.tensor(r, dtype=torch.int64)
    flat = flat.cuda()
    st["table"] = torch.where(flat >= 0, order[flat.clamp(min=0)], -1).int().contiguous()
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["groups"] = torch.tensor([0] + sizes, device="cuda").cumsum(0).int()
    st["shared"] = torch.tensor(shared, dtype=torch.int32, device="cuda")
    st["q"] = torch.randn(len(lens), case["heads"], dim, device="cuda",
                          generator=gen).to(_TYPES[case["type"]])
    st["k_scale"] = st["v_scale"] = None
    if case["kv"] == "e4m3":
        st["k_scale"], st["v_scale"] = (torch.rand(hkv, device="cuda", generator=gen) * 0.5 + 0.75
                                        for _ in range(2))
    st["scale"], st["lse"], st["page"] = dim ** -0.5, case["lse"], page


def _prepare_sample(case, gen, st) -> None:
    rows, vocab = case["rows"], case["vocab"]
    # a language model's logits: a few likely tokens whose probabilities fall like a power of
    # their rank, and a wide body far below them
    x = 2 * torch.randn(rows, vocab, device="cuda", generator=gen) - 4
    top = min(vocab, 64)
    at = torch.rand(rows, vocab, device="cuda", generator=gen).topk(top, -1).indices
    peak = 12 - 2 * torch.log(1.0 + torch.arange(top, device="cuda"))
    noise = 0.5 * torch.randn(rows, top, device="cuda", generator=gen)
    st["logits"] = x.scatter(1, at, peak + noise).to(_TYPES[case["type"]])
    st["u"] = torch.rand(rows, device="cuda", generator=gen)
    st["temperature"], st["top_k"] = case["temperature"], case["top_k"]
    st["top_p"], st["min_p"] = case["top_p"], case["min_p"]
    if case["how"] == "rows":                                # settings of each request
        rng = random.Random(case["mix"])
        t, k, p, m = [], [], [], []
        for _ in range(rows):
            t.append(rng.choice((0.0, 0.7, 1.0, case["temperature"])))
            k.append(rng.choice((0, case["top_k"], case["top_k"])))
            p.append(rng.choice((1.0, case["top_p"], case["top_p"])))
            m.append(rng.choice((0.0, 0.0, case["min_p"])))
        st["temperature"], st["top_p"], st["min_p"] = (
            torch.tensor(z, dtype=torch.float32, device="cuda") for z in (t, p, m))
        st["top_k"] = torch.tensor(k, dtype=torch.int32, device="cuda")


def _prepare_rotary(case, gen, st) -> None:
    rows, heads, hkv, dim = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    typ = _TYPES[case["type"]]
    cols = (heads + 2 * hkv) * dim
    buf = torch.randn(rows, cols + case["pad"], device="cuda", generator=gen).to(typ)[:, :cols]
    st["q"] = buf[:, :heads * dim].unflatten(1, (heads, dim))
    st["k"] = buf[:, heads * dim:(heads + hkv) * dim].unflatten(1, (hkv, dim))
    first = max(0, case["far"] - rows)
    at = first + torch.arange(rows, device="cuda") % max(1, case["far"] - first)
    if case["pads"]:
        at[max(0, rows - case["pads"]):] = -1
    st["positions"] = at
    half = case["turned"] // 2
    t = torch.arange(half, device="cuda", dtype=torch.float64)
    st["freqs"] = THETA ** (-2 * t / case["turned"])
    if case["amplitude"] != 1.0:                             # scaled: long waves eight times longer
        st["freqs"] = torch.where(st["freqs"] < 2 * math.pi / 4096, st["freqs"] / 8, st["freqs"])
    st["q_norm"] = st["k_norm"] = None
    if case["norm"]:
        st["q_norm"], st["k_norm"] = (
            (1 + 0.05 * torch.randn(dim, device="cuda", generator=gen)).to(typ) for _ in range(2))
    st["interleaved"], st["amplitude"] = case["interleaved"], case["amplitude"]


# ------------------------------------------------------------------------------ one pass
_package = None


def _framework():
    global _package
    if _package is None:
        import __graft_entry__

        _package = __graft_entry__.import_package()
        import moss_tts_lite_amd.paged
        import moss_tts_lite_amd.rotary
        import moss_tts_lite_amd.sampling
    return _package


def run(st):
    if st["kind"] == "shared":
        return _own_shared(st) if own else _shared(st)
    if st["kind"] == "sample":
        return _own_sample(st) if own else _sample(st)
    return _own_rotary(st) if own else _rotary(st)


def _own_shared(st):
    got = _framework().paged.paged_attention_shared(
        st["q"], st["k"], st["v"], st["table"], st["lens"], st["groups"], st["shared"],
        st["scale"], st["k_scale"], st["v_scale"], return_lse=st["lse"])
    return {"out": got[0], "lse": got[1]} if st["lse"] else {"out": got}


def _own_sample(st):
    token, logprob = _framework().sampling.sample(
        st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"],
        return_logprob=True)
    return {"token": token, "logprob": logprob}


def _own_rotary(st):
    q, k = _framework().rotary.qk_rotary(
        st["q"], st["k"], st["positions"], st["freqs"], st["q_norm"], st["k_norm"], eps=EPS,
        interleaved=st["interleaved"], amplitude=st["amplitude"])
    return {"q": q, "k": k}


# ------------------------------------------------------------------------------ plain forms
def _shared(st):
    """Every sequence over all of its own pages."""
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
    keep = torch.arange(k.shape[2], device=q.device)[None] < lens[:, None]
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


def _rows_of(x, like) -> torch.Tensor:
    """A setting for all rows, or one for each, as float64 [rows, 1]."""
    if not isinstance(x, torch.Tensor):                      # a number is a float32 setting too
        x = torch.full((like.shape[0],), x, dtype=torch.float32, device=like.device)
    return x.double()[:, None]


def _sample(st):
    """Sums in float64: a token differs where a sum is off by more than u lies from a border, and
    a row has as many borders as tokens."""
    x = st["logits"].double()
    t, k, p, m = (_rows_of(st[n], x) for n in ("temperature", "top_k", "top_p", "min_p"))
    x = torch.where(torch.isnan(x), float("-inf"), x)
    sx, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = sx[:, :1]
    rank = torch.arange(x.shape[1], device=x.device)[None]
    k = torch.where((k <= 0) | (k > x.shape[1]), x.shape[1], k)
    w = torch.where(sx == top, 1.0, torch.exp((sx - top) / torch.where(t > 0, t, 1.0)))
    w = torch.where(sx == float("-inf"), 0.0, w)
    w = torch.where(t > 0, w, (rank == 0).double())          # greedy: the first of the order
    wk = torch.where(rank < k, w, 0.0)
    upto = wk.cumsum(-1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], -1)
    keep = (rank < k) & (w > 0) & ((before <= p * upto[:, -1:]) | (p >= 1)) & (w >= m)
    keep[:, :1] = True
    at = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))
    c = at.cumsum(-1)
    total = c[:, -1:]
    token = (c <= st["u"].double()[:, None] * total).sum(-1, keepdim=True)
    last = torch.where(at > 0, rank, -1).amax(-1, keepdim=True)
    token = torch.minimum(token, last).clamp(min=0)
    logprob = torch.log(at.gather(1, token) / total)
    none = top == float("-inf")
    return {"token": torch.where(none, -1, token)[:, 0],
            "logprob": torch.where(none, float("-inf"), logprob)[:, 0].float()}


def _rotary(st):
    typ = st["q"].dtype
    ang = st["positions"].double()[:, None] * st["freqs"]    # 64 bits: far positions
    c, s = ((f(ang) * st["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    there = (st["positions"] >= 0)[:, None, None]

    def one(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        half = c.shape[-1]
        part, rest = x[..., :2 * half], x[..., 2 * half:]
        if st["interleaved"]:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        else:
            a, b = part[..., :half], part[..., half:]
            part = torch.cat([a * c - b * s, b * c + a * s], -1)
        return torch.where(there, torch.cat([part, rest], -1), 0.0).to(typ)

    return {"q": one(st["q"], st["q_norm"]), "k": one(st["k"], st["k_norm"])}


# ------------------------------------------------------------------------------ work
def work(case) -> dict:
    if case["kind"] == "shared":
        dim, hkv, heads = case["dim"], case["kv_heads"], case["heads"]
        size = 1 if case["kv"] == "e4m3" else 2
        sizes, shared, lens = _layout(case)
        at, read = 0, 0
        for n, s in zip(sizes, shared):
            mine = lens[at:at + n]
            at += n
            read += min(s, max(mine)) + sum(max(0, x - s) for x in mine)
        return {"bytes": 2 * read * hkv * dim * size + 4 * len(lens) * heads * dim
                + 4 * (read // case["page"] + 2 * len(lens))
                + (4 * len(lens) * heads if case["lse"] else 0),
                "flops": 4 * sum(lens) * heads * dim}
    if case["kind"] == "sample":
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * size + 16), "flops":
                4 * case["rows"] * case["vocab"]}
    n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
    return {"bytes": 4 * n + 8 * case["rows"] + 4 * case["turned"], "flops": 10 * n}


# ------------------------------------------------------------------------------ definitions
def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "shared":
        return _exact_shared(st)
    return _exact_sample(st) if st["kind"] == "sample" else _exact_rotary(st)


def _exact_shared(st):
    """Sequence by sequence over exactly its positions, in float64."""
    q, page = st["q"].double(), st["page"]
    b, heads, dim = q.shape
    hkv = st["k"].shape[1]
    g = heads // hkv
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
            at = slice(h * g, (h + 1) * g)
            s = (k @ q[i, at].T).T * st["scale"]
            lse[i, at] = torch.logsumexp(s, -1)
            out[i, at] = torch.softmax(s, -1) @ v
    return {"out": out, "lse": lse} if st["lse"] else {"out": out}


def _exact_sample(st):
    """Row by row on the host: the kept tokens by their order, then the draw by index."""
    rows, vocab = st["logits"].shape
    tokens, logs = [], []

    def setting(name, i):
        x = st[name]
        return float(x[i]) if isinstance(x, torch.Tensor) else float(np.float32(x))

    for i in range(rows):
        x = st["logits"][i].double().cpu().numpy()
        t, k, p, m = (setting(n, i) for n in ("temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-x, kind="stable")
        if t <= 0:
            tokens.append(int(order[0]))
            logs.append(0.0)
            continue
        if 0 < k < vocab:
            order = order[:int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        n = len(order)
        if p < 1:
            n = max(1, int(np.searchsorted(np.concatenate([[0.0], np.cumsum(w)[:-1]]),
                                           p * np.sum(w), side="right")))
        n = max(1, min(n, int((w >= m).sum())))
        kept = np.sort(order[:n])
        w = np.exp((x[kept] - x[order[0]]) / t)
        c = np.cumsum(w)
        j = min(int(np.searchsorted(c, float(st["u"][i]) * c[-1], side="right")), n - 1)
        tokens.append(int(kept[j]))
        logs.append(float(np.log(w[j] / c[-1])))
    return {"token": torch.tensor(tokens), "logprob": torch.tensor(logs, dtype=torch.float64)}


def _exact_rotary(st):
    pos = st["positions"].double()
    half = st["freqs"].numel()
    turn = torch.polar(torch.full((), st["amplitude"], dtype=torch.float64, device=pos.device)
                       .expand(len(pos), half).contiguous(), pos[:, None] * st["freqs"])[:, None]
    got = {}
    for name in ("q", "k"):
        x, w = st[name].double(), st[name + "_norm"]
        if w is not None:
            x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
        a, b = (x[..., :2 * half:2], x[..., 1:2 * half:2]) if st["interleaved"] else (
            x[..., :half], x[..., half:2 * half])
        z = torch.complex(a.contiguous(), b.contiguous()) * turn
        y = x.clone()
        if st["interleaved"]:
            y[..., :2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
        else:
            y[..., :half], y[..., half:2 * half] = z.real, z.imag
        y[st["positions"] < 0] = 0
        got[name] = y
    return got
