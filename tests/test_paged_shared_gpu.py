"""Attention of sequences that share a prefix against float64 over each sequence's own pages, and a
step of forks through rotation, write, attention and draw together."""
import random

import pytest
import torch

from moss_tts_lite_amd import paged, rotary, sampling
from tests._paged import HALF_STEP, TYPES, attention64
from tests._paged_numbers import beside, coded_case, room, sink_case
from tests._sampling import reference as sample_reference

pytestmark = pytest.mark.gpu


def shared_case(dev, sizes, shared, lens, H, Hkv, D, page, typ="bf16", kv="bf16", seed=0, room=33):
    """Groups whose whole shared pages are held by all, and whose partly shared page is copied; pages
    and rows that nobody holds are NaN.  ``room``: entries of the table past the longest sequence;
    tables of more than 512 positions are the ones whose prefixes are read once."""
    gen = torch.Generator().manual_seed(seed)
    width = max([1] + [-(-n // page) for n in lens]) + room
    need = sum(-(-n // page) for n in lens) + sum(s // page for s in shared) + 3
    order = torch.randperm(need, generator=gen).tolist()
    pool = torch.full((2, need, Hkv, page, D), float("nan"))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for n, s in zip(sizes, shared):
        most = max([0] + lens[at:at + n])
        prefix = torch.randn(2, Hkv, s, D, generator=gen)
        trunk = [order.pop() for _ in range(min(s, most) // page)]
        for j, p in enumerate(trunk):
            pool[:, p] = prefix[:, :, j * page:(j + 1) * page]
        for i in range(at, at + n):
            for j in range(-(-lens[i] // page)):
                if j < len(trunk):
                    table[i, j] = trunk[j]
                    continue
                p = order.pop()
                table[i, j] = p
                rows = min(page, lens[i] - j * page)
                pool[:, p, :, :rows] = torch.randn(2, Hkv, rows, D, generator=gen)
                same = min(max(s - j * page, 0), rows)
                pool[:, p, :, :same] = prefix[:, :, j * page:j * page + same]
        at += n
    scales = [torch.rand(Hkv, generator=gen) + 0.5 if kv == "e4m3" else None for _ in range(2)]
    starts = torch.tensor([0] + list(sizes)).cumsum(0).int()
    q = torch.randn(len(lens), H, D, generator=gen).to(TYPES[typ])
    pool = pool.to(TYPES[kv])
    t = [x if x is None else x.to(dev) for x in (
        q, pool[0], pool[1], table, torch.tensor(lens, dtype=torch.int32), starts,
        torch.tensor(shared, dtype=torch.int32), *scales)]
    return dict(q=t[0], k_pages=t[1], v_pages=t[2], table=t[3], lens=t[4], groups=t[5], shared=t[6],
                scale=D ** -0.5, k_scale=t[7], v_scale=t[8])


def check(a):
    out, lse = paged.paged_attention_shared(**a, return_lse=True)
    alone = {k: v for k, v in a.items() if k not in ("groups", "shared")}
    ref, rlse, mag = attention64(**alone)
    got = out.cpu().double()
    assert not got.isnan().any()
    # the output's rounding; weights in two terms (2^-16) and float32 scores: D products of
    # |q k| scale, about 8 in all, each 2^-24 off per sum step (under 2^-14)
    tol = HALF_STEP[out.dtype] * ref.abs() + (2 ** -16 + 2 ** -14) * mag + 2.0 ** -24
    worst = ((got - ref).abs() - tol).max() if got.numel() else torch.tensor(-1.0)
    assert float(worst) <= 0, float(worst)
    empty = rlse == float("-inf")
    assert torch.equal(lse.cpu() == float("-inf"), empty)
    if (~empty).any():
        assert float((lse.cpu().double() - rlse)[~empty].abs().max()) < 2e-4
    return out


OWN = [0, 1, 2, 15, 16, 17, 33, 127, 128, 129]
SHARED = [0, 1, 15, 16, 17, 31, 32, 33, 47, 127, 128, 129, 160, 300]


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_edges(dev, page, kv):
    rng = random.Random(page)
    sizes = [rng.randint(2, 5) for _ in SHARED]
    lens = [s + rng.choice(OWN) for n, s in zip(sizes, SHARED) for _ in range(n)]
    check(shared_case(dev, sizes, SHARED, lens, 8, 2, 128, page, "bf16", kv, page))


@pytest.mark.parametrize("H,Hkv", [(1, 1), (4, 4), (7, 1), (28, 4), (16, 1), (17, 1), (40, 2),
                                   (96, 2), (65, 1), (130, 1), (32, 8)])
@pytest.mark.parametrize("typ,kv,D", [("bf16", "bf16", 128), ("f16", "f16", 64),
                                      ("f16", "e4m3", 128), ("bf16", "e4m3", 64)])
def test_heads_and_types(dev, H, Hkv, typ, kv, D):
    check(shared_case(dev, [3, 1, 4], [200, 30, 77], [210, 200, 333, 90, 77, 78, 0, 150], H, Hkv, D,
                      16, typ, kv, H))


# tables of up to 512 positions: 512 sequences times kv heads and sets of 16 query heads, and more
@pytest.mark.parametrize("n,H,Hkv", [(3, 8, 2), (63, 28, 4), (64, 32, 8), (65, 32, 8), (255, 34, 2),
                                     (300, 17, 1)])
@pytest.mark.parametrize("typ,kv,D,page", [("bf16", "bf16", 128, 16), ("f16", "e4m3", 64, 32),
                                           ("f16", "f16", 128, 256)])
def test_short_tables(dev, n, H, Hkv, typ, kv, D, page):
    rng = random.Random(n)
    shared = [rng.choice([0, 17, 64, 300]) for _ in range(n // 3)]
    lens = [min(s + rng.choice(OWN), 512) if rng.random() < .9 else 0
            for s in shared for _ in range(3)]
    check(shared_case(dev, [3] * (n // 3), shared, lens, H, Hkv, D, page, typ, kv, n, 0))


@pytest.mark.parametrize("room", [0, 1])
def test_tables_of_512_and_more(dev, room):
    check(shared_case(dev, [3, 1], [300, 0], [300, 512, 0, 470], 8, 2, 128, 16, room=room))


# 1 to 5 sets of 16 columns, and columns that end inside one
@pytest.mark.parametrize("n,H,Hkv", [(2, 1, 1), (2, 8, 1), (3, 8, 1), (2, 16, 1), (4, 12, 1),
                                     (5, 13, 1), (9, 7, 1), (16, 4, 1), (17, 4, 1), (70, 2, 2)])
@pytest.mark.parametrize("shared", [40, 700, 2100])
def test_columns(dev, n, H, Hkv, shared):
    rng = random.Random(n + shared)
    check(shared_case(dev, [n], [shared], [shared + rng.randint(0, 300) for _ in range(n)], H, Hkv,
                      128, 32, seed=n))


@pytest.mark.parametrize("sizes,shared", [([1], [500]), ([1, 1, 1], [9, 600, 0]),
                                          ([5, 0, 3, 1], [600, 50, 1100, 20]),
                                          ([2] * 30, [16 * i for i in range(30)]),
                                          ([1, 40, 2], [0, 1500, 90])])
def test_groups(dev, sizes, shared):
    rng = random.Random(len(sizes))
    lens = [s + rng.randint(0, 200) for n, s in zip(sizes, shared) for _ in range(n)]
    check(shared_case(dev, sizes, shared, lens, 8, 2, 128, 16, seed=len(sizes)))


def test_short_and_empty_sequences(dev):
    # sequences that end inside the shared positions, finished ones, a group of finished ones
    lens = [0, 300, 10, 0, 299, 0, 0, 1, 700, 0, 20, 64, 33]
    a = shared_case(dev, [5, 2, 2, 3, 1], [290, 50, 400, 60, 9], lens, 8, 2, 128, 16, seed=3)
    check(a)
    a["shared"] = torch.tensor([100000, 50, -5, 2 ** 31 - 1, 7], dtype=torch.int32, device=dev)
    a["lens"][:] = torch.tensor([0, 288, 10, 0, 150, 0, 0, 1, 700, 0, 20, 60, 33])
    # no two of a group may now differ in what they hold before the group's longest end
    a["shared"][0], a["shared"][3] = 288, 16
    check(a)
    none = shared_case(dev, [3], [100], [0, 0, 0], 8, 2, 128, 16)
    assert not check(none).any()
    a = {k: v[:0] if k in ("q", "table", "lens", "shared") else v[:1] if k == "groups" else v
         for k, v in none.items()}
    assert paged.paged_attention_shared(**a).shape == (0, 8, 128)


def test_no_sequence_reaches_the_shared_positions(dev):
    # read through the longest, and no further
    a = shared_case(dev, [4], [500], [100, 230, 0, 17], 8, 2, 128, 16, seed=5)
    check(a)


def test_sequences_outside_the_groups(dev):
    a = shared_case(dev, [2, 3, 2], [80, 200, 40], [90, 85, 210, 200, 333, 41, 50], 8, 2, 64, 16)
    a["groups"], a["shared"] = a["groups"][1:3].contiguous(), a["shared"][1:2].contiguous()
    check(a)
    a["groups"], a["shared"] = a["groups"][:1].contiguous(), a["shared"][:0].contiguous()
    check(a)


@pytest.mark.parametrize("n", [6, 300, 600])     # sequences in LDS or not
@pytest.mark.parametrize("repeats", [1, 250, 600])
def test_groups_that_do_not_ascend(dev, n, repeats):
    """Overlapping groups are not there: each sequence is attended by itself."""
    rng = random.Random(n)
    a = shared_case(dev, [n], [64], [rng.choice([0, 64, 65, 200]) for _ in range(n)], 8, 2, 64, 16,
                    room=40)
    want = None
    for starts in ([0, n] * repeats, [n, 0] * repeats, [0, 2, 1] + [n] * repeats,
                   [0, 2 ** 31 - 1, -(2 ** 31)] * repeats, [0] * repeats + [n, n - 1]):
        a["groups"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        if (a["groups"][1:] >= a["groups"][:-1]).all():
            continue
        a["shared"] = torch.full((len(starts) - 1,), 64, dtype=torch.int32, device=dev)
        if want is None:
            want = check(a)
        assert torch.equal(paged.paged_attention_shared(**a), want)
    # numbers past the batch are its ends
    a["groups"] = torch.tensor([-5, n + 3, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    a["shared"] = torch.full((2,), 64, dtype=torch.int32, device=dev)
    check(a)


def test_holes_and_long_lens(dev):
    a = shared_case(dev, [3], [128], [140, 200, 170], 8, 2, 128, 16, seed=4)
    a["table"][:, 2] = -1                            # a hole in the shared pages
    a["table"][:, 5] = a["k_pages"].shape[0]
    a["table"][1, 9] = -7                            # and in one's own
    check(a)
    for x in ("k_pages", "v_pages"):                 # rows behind a length are attended to now
        a[x] = a[x].nan_to_num()
    a["lens"] += 100000                              # past the table: holes up to its width
    check(a)
    a["lens"][:] = torch.tensor([-3, -(1 << 31), 140])
    check(a)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.5, -2.0])
def test_scales_of_either_sign(dev, kv, scale):
    a = shared_case(dev, [3, 20], [500, 300], [520, 500, 640] + [300 + i for i in range(20)], 8, 2,
                    64, 16, "bf16", kv, 12)
    a["scale"] = scale
    if kv == "e4m3":
        a["k_scale"][1] *= -1
        a["v_scale"][0] *= -1
    # scores are up to 12 times larger here: so is what float32 products are off
    out, lse = paged.paged_attention_shared(**a, return_lse=True)
    ref, rlse, mag = attention64(**{k: v for k, v in a.items() if k not in ("groups", "shared")})
    rel = 2 ** -16 + 2 ** -14 * max(1, abs(scale) * 8)
    assert ((out.cpu().double() - ref).abs() <= 2 ** -8 * ref.abs() + rel * mag + 2.0 ** -24).all()
    assert ((lse.cpu().double() - rlse).abs() <= 2e-4 * max(1, abs(scale) * 8)).all()


@pytest.mark.parametrize("n", [511, 512, 513])
def test_as_many_sequences_as_fit_a_workgroups_lists(dev, n):
    sizes = [7] * (n // 7) + ([n % 7] if n % 7 else [])
    rng = random.Random(n)
    shared = [rng.choice([0, 48, 400]) for _ in sizes]
    lens = [s + rng.randint(0, 40) for k, s in zip(sizes, shared) for _ in range(k)]
    check(shared_case(dev, sizes, shared, lens, 2, 1, 64, 16, seed=n))


def test_more_groups_than_sequences(dev):
    sizes = [0] * 300 + [3] + [0] * 300 + [2]
    shared = [50] * 300 + [600] + [9] * 300 + [700]
    check(shared_case(dev, sizes, shared, [610, 600, 777, 700, 730], 8, 2, 128, 16, seed=9))


# 64 query heads to a kv head and more: a sequence is whole items of 64 columns, several of a lane's
# run of sequences, and some have nothing of their own
@pytest.mark.parametrize("n", [65, 96, 192])
@pytest.mark.parametrize("H,Hkv", [(64, 1), (71, 1), (128, 1), (128, 2), (512, 8)])
@pytest.mark.parametrize("grouped", [False, True])
def test_many_sequences_of_wide_heads(dev, n, H, Hkv, grouped):
    rng = random.Random(n + H)
    sizes, shared, lens = [], [], []
    while len(lens) < n:
        m = min(rng.randint(1, 12) if grouped else 1, n - len(lens))
        s = rng.choice([0, 40, 128, 260, 300]) if grouped else 0
        sizes.append(m)
        shared.append(s)
        for _ in range(m):
            r = rng.random()
            lens.append(0 if r < .15 else rng.randint(0, s) if r < .3 else
                        s + rng.choice([1, 100, 128, 129, 300, 640]))
    check(shared_case(dev, sizes, shared, lens, H, Hkv, 64, 16, seed=n))


def test_growing_and_falling_scores(dev):
    # the running maximum moves in every tile, or never after the first
    for sign in (1, -1):
        a = shared_case(dev, [20], [2000], [2000 + 5 * i for i in range(20)], 8, 2, 128, 32, seed=3)
        n, hkv, page, d = a["k_pages"].shape
        rank = torch.full((n,), 0.0, device=dev)
        rank[a["table"][0, :62].long()] = torch.arange(62, device=dev).float()
        a["k_pages"] = (a["k_pages"].nan_to_num() * 0.05).float()
        a["k_pages"][..., 0] += sign * rank[:, None, None] * 0.5
        a["k_pages"] = a["k_pages"].bfloat16()
        a["v_pages"] = a["v_pages"].nan_to_num()
        a["q"][..., 0] = 8.0                         # a page's scores are some 0.35 above the last's
        out = paged.paged_attention_shared(**a)
        ref, _, mag = attention64(**{k: v for k, v in a.items() if k not in ("groups", "shared")})
        # scores up to 22: 2^-24 of the products' sizes (some 260) a step
        assert ((out.cpu().double() - ref).abs() <=
                2 ** -8 * ref.abs() + (2 ** -16 + 2 ** -12) * mag + 2.0 ** -24).all()


def test_many_sequences(dev):
    rng = random.Random(1)
    sizes = [rng.randint(1, 30) for _ in range(90)]  # past what a workgroup keeps of lengths
    while sum(sizes) <= 1100:
        sizes.append(rng.randint(1, 30))
    shared = [rng.choice([0, 16, 33, 90, 200]) for _ in sizes]
    lens = [s + rng.randint(0, 60) for n, s in zip(sizes, shared) for _ in range(n)]
    check(shared_case(dev, sizes, shared, lens, 4, 2, 64, 16, seed=2))


def test_long_prefixes(dev):
    check(shared_case(dev, [6, 2], [20000, 9000], [20001, 20500, 20000, 21000, 0, 20100, 9100, 9000],
                      8, 2, 128, 64, seed=6))
    check(shared_case(dev, [30], [5000], [5000 + 7 * i for i in range(30)], 4, 1, 64, 32, "f16",
                      "f16", seed=7))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_layouts(dev, kv):
    a = shared_case(dev, [3, 2], [100, 64], [130, 100, 177, 90, 64], 8, 2, 128, 32, "bf16", kv, 8)
    want = check(a)
    b = dict(a)
    for x in ("k_pages", "v_pages"):                 # tokens before heads; rows further apart
        n, hkv, page, d = a[x].shape
        wide = torch.zeros(n, page, hkv, d + 32, dtype=a[x].dtype, device=dev)
        wide[..., :d] = a[x].transpose(1, 2)
        b[x] = wide[..., :d].transpose(1, 2)
    assert torch.equal(paged.paged_attention_shared(**b), want)
    qkv = torch.randn(5, 12 * 128, device=dev).bfloat16()
    qkv[:, 128:128 * 9] = a["q"].flatten(1)
    b["q"] = qkv[:, 128:128 * 9].unflatten(1, (8, 128))
    assert torch.equal(paged.paged_attention_shared(**b), want)
    b["q"] = a["q"].transpose(0, 2).contiguous().transpose(0, 2)       # no adjacent dims: copied
    assert torch.equal(paged.paged_attention_shared(**b), want)


def test_past_32_bit_offsets(dev):
    pages, Hkv, page, D = 140000, 1, 128, 128        # 2.3e9 elements of K and of V
    k = torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    held = [0, 139999, 131072, 70001, 139000]
    for p in held:
        k[p], v[p] = (torch.randn(Hkv, page, D, device=dev).bfloat16() for _ in range(2))
    table = torch.tensor([[139999, 131072, 0], [139999, 131072, 70001], [139999, 131072, 139000]],
                         dtype=torch.int32, device=dev)
    a = dict(q=torch.randn(3, 4, D, device=dev).bfloat16(), k_pages=k, v_pages=v, table=table,
             lens=torch.tensor([300, 384, 257], dtype=torch.int32, device=dev), scale=D ** -0.5,
             groups=torch.tensor([0, 3], dtype=torch.int32, device=dev),
             shared=torch.tensor([256], dtype=torch.int32, device=dev))
    got = paged.paged_attention_shared(**a)
    b = {k_: v_ for k_, v_ in a.items() if k_ not in ("groups", "shared")}
    small = {p: i for i, p in enumerate(held)}
    b["k_pages"], b["v_pages"] = k[held], v[held]
    b["table"] = torch.tensor([[small[int(x)] for x in r] for r in table.tolist()],
                              dtype=torch.int32)
    ref, _, mag = attention64(**b)
    tol = 2 ** -8 * ref.abs() + (2 ** -16 + 2 ** -14) * mag + 2.0 ** -24
    assert ((got.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("typ,kv,D", [("bf16", "bf16", 128), ("f16", "f16", 64),
                                      ("bf16", "e4m3", 64), ("f16", "e4m3", 128)])
@pytest.mark.parametrize("lens,sizes,shared", [([700, 690, 800], [3], [640]),
                                               ([65, 64, 33, 40], [2, 2], [64, 32]),
                                               ([3000] * 5, [5], [2999]), ([513] * 20, [20], [512])])
@pytest.mark.parametrize("code", ["position", "tile"])
def test_weights_to_the_rounding(dev, typ, kv, D, lens, sizes, shared, code):
    # V that codes its row: a lost, doubled or misplaced row shows, whatever the tolerance
    args, (ref, rlse) = coded_case(lens, 8, 2, D, 16, typ, kv, code)
    a = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    i32 = dict(dtype=torch.int32, device=dev)
    out, lse = paged.paged_attention_shared(
        **a, groups=torch.tensor([0] + sizes, device=dev).cumsum(0).int(),
        shared=torch.tensor(shared, **i32), return_lse=True)
    n = max(lens)
    assert not beside(out.cpu(), ref, room(n, typ, 4)).any()
    assert ((lse.cpu().double() - rlse).abs() <= room(n, typ, 4) + 2 ** -22 * rlse.abs()).all()


@pytest.mark.parametrize("typ,kv,D,c", [("bf16", "bf16", 128, 8.0), ("f16", "f16", 64, 8.0),
                                        ("f16", "f16", 128, 12.0), ("bf16", "e4m3", 128, 8.0)])
def test_small_weights_beside_a_large_one(dev, typ, kv, D, c):
    args, (ref, _) = sink_case([900, 700, 640], 8, 2, D, 16, typ, kv, c)
    a = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    i32 = dict(dtype=torch.int32, device=dev)
    out = paged.paged_attention_shared(**a, groups=torch.tensor([0, 3], **i32),
                                       shared=torch.tensor([640], **i32))
    assert not beside(out.cpu(), ref, room(900, typ, 1.875 * c)).any()


def test_repeats_bitwise_captures_and_streams(dev):
    a = shared_case(dev, [6, 1, 3], [900, 0, 300], [900 + 30 * i for i in range(6)] +
                    [50] + [300, 777, 0], 32, 8, 128, 16, seed=11)
    want = paged.paged_attention_shared(**a, return_lse=True)
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = paged.paged_attention_shared(**a, return_lse=True)
        graphs.append((g, res, torch.cuda.Stream()))
    for _ in range(4):
        for g, res, s in graphs:
            with torch.cuda.stream(s):
                res[0].fill_(7)
                g.replay()
        again = paged.paged_attention_shared(**a)    # eager at the same time
        torch.cuda.synchronize()
        assert torch.equal(again, want[0])
        for _, res, _ in graphs:
            assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
    a["lens"][3], a["lens"][8], a["shared"][0] = 905, 301, 800            # the step moves on
    for g, res, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], check(a))


@pytest.mark.parametrize("typ,kv", [("bf16", "e4m3"), ("f16", "f16"), ("f16", "e4m3")])
def test_the_same_call_gives_the_same_bits(dev, typ, kv):
    a = shared_case(dev, [20, 2, 40], [3000, 300, 777], [3000 + 40 * i for i in range(20)] +
                    [300, 0] + [777 + 9 * i for i in range(40)], 32, 8, 128, 32, typ, kv, seed=13)
    want = paged.paged_attention_shared(**a, return_lse=True)
    for _ in range(30):
        got = paged.paged_attention_shared(**a, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_schemas(dev):
    from moss_tts_lite_amd import ops

    a = shared_case(dev, [2], [64], [80, 64], 8, 2, 64, 16)
    for x in ("k_pages", "v_pages"):
        a[x] = a[x].nan_to_num()                     # compared as values
    args = tuple(a[x] for x in ("q", "k_pages", "v_pages", "table", "lens", "groups", "shared",
                                "scale"))
    for name in ("paged_attention_shared", "paged_attention_shared_lse"):
        torch.library.opcheck(ops.overload(name), args, test_utils=("test_schema",
                                                                    "test_faketensor"))


# ------------------------------------------------------------------------------ together
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_step_of_forks(dev, captured, interleaved):
    """Prompts, forks, then steps: rows are rotated in place, written into pages, attended with the
    shared prefix read once, and each candidate's token is drawn."""
    H, Hkv, D, page, turned, vocab = 8, 2, 64, 16, 32, 500
    gen = torch.Generator().manual_seed(3)
    k, v, table, lens, refs = paged.new_cache(1, 60, Hkv, page, D, 9, 12)
    freqs = rotary.rotary_freqs(turned, 1e4, 4.0, original=64)
    amp = rotary.rotary_amplitude(4.0)
    head = torch.randn(H * D, vocab, generator=gen).to(dev) / 8
    cols = (H + 2 * Hkv) * D
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    rows = {}

    def rotated(x, pos):
        """The row's q, k, v in float64, k and v as the pages hold them."""
        y = x.cpu().double().view(-1, D).clone()
        for h in range(H + Hkv):
            for t in range(turned // 2):
                i, j = (2 * t, 2 * t + 1) if interleaved else (t, t + turned // 2)
                z = torch.polar(torch.tensor(amp).double(), pos * freqs[t].cpu())
                z = complex(y[h, i], y[h, j]) * complex(z)
                y[h, i], y[h, j] = z.real, z.imag
        y = y.bfloat16().double()
        return y[:H], y[H:H + Hkv], y[H + Hkv:]

    def rotate(x, at):
        q, kk, _ = x.split([H * D, Hkv * D, Hkv * D], 1)
        rotary.qk_rotary_(q.unflatten(1, (H, D)), kk.unflatten(1, (Hkv, D)), at, freqs,
                          interleaved=interleaved, amplitude=amp)

    prompts = {0: 37, 1: 64}
    for s, n in prompts.items():
        paged.check(paged.pages_extend(table, lens, refs, ints([s]), ints([n]), k, v))
        x = torch.randn(n, cols, generator=gen).bfloat16().to(dev)
        for p in range(n):
            rows[s, p] = rotated(x[p], p)
        at = torch.arange(n, device=dev)
        rotate(x, at)
        paged.paged_write(x, k[0], v[0], table, at, ints([s] * n))
    kids = {0: [2, 3, 4], 1: [5, 6]}
    for s, c in kids.items():
        paged.check(paged.pages_fork(table, lens, refs, ints([s] * len(c)), ints(c), page))
        for i in c:
            rows.update({(i, p): rows[s, p] for p in range(prompts[s])})
    seqs = ints([0, 2, 3, 4, 1, 5, 6])               # each prompt beside its forks
    groups, shared = ints([0, 4, 7]), ints([37, 64])
    n = len(seqs)
    buf = torch.zeros(n, cols, dtype=torch.bfloat16, device=dev)
    u = torch.zeros(n, device=dev)

    def step():
        status = paged.pages_extend(table, lens, refs, seqs, torch.ones_like(seqs), k, v)
        mine, length = table[seqs], lens[seqs]
        at = torch.where(status == 0, length.long() - 1, -1)
        rotate(buf, at)
        q = paged.paged_write(buf, k[0], v[0], mine, at)
        out = paged.paged_attention_shared(q, k[0], v[0], mine, length, groups, shared, D ** -0.5)
        logits = out.flatten(1).float() @ head
        return status, out, logits, sampling.sample(logits, u, 0.8, top_k=40, top_p=0.9)

    graph = None
    if captured:
        state = [x.clone() for x in (table, lens, refs, k, v)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):                   # the library product's own set-up
            step()
        torch.cuda.current_stream().wait_stream(s)
        for x, y in zip((table, lens, refs, k, v), state):
            x.copy_(y)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for x, y in zip((table, lens, refs, k, v), state):
            x.copy_(y)
    for _ in range(6):
        x = torch.randn(n, cols, generator=gen).bfloat16()
        r = torch.rand(n, generator=gen)
        pos = [int(lens[int(s)]) for s in seqs]
        for i, s in enumerate(seqs.tolist()):
            rows[s, pos[i]] = rotated(x[i], pos[i])
        buf.copy_(x)
        u.copy_(r)
        if graph:
            graph.replay()
        else:
            got = step()
        status, out, logits, token = got
        paged.check(status)
        for i, s in enumerate(seqs.tolist()):
            kk = torch.stack([rows[s, p][1] for p in range(pos[i] + 1)])
            vv = torch.stack([rows[s, p][2] for p in range(pos[i] + 1)])
            g = H // Hkv
            sc = torch.einsum("hd,phd->hp", rows[s, pos[i]][0],
                              kk.repeat_interleave(g, 1)) * D ** -0.5
            ref = torch.einsum("hp,phd->hd", torch.softmax(sc, -1), vv.repeat_interleave(g, 1))
            err = (out[i].double().cpu() - ref).norm() / ref.norm()
            # roundings of 2^-9 in q, k, v and the output, which float32 may take the other way
            assert float(err) < 1e-2, (s, pos[i], float(err))
        for i, (tok, _, near) in enumerate(sample_reference(logits, u, 0.8, 40, 0.9)):
            assert near > 2 ** -30 and int(token[i]) == tok
