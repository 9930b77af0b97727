"""The paged cache on the device where a call goes past the usual: refused bookkeeping calls with
wild arguments, compared with everything around the state they must leave alone, and the documented
decode step when its extend is refused."""
import textwrap

import pytest
import torch

from moss_tts_lite_amd import paged
from tests._paged import Pages

pytestmark = pytest.mark.gpu

PAGE = 16


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------ refused calls
class Guarded:
    """Sequences in the middle of larger buffers, so that a write beside the state shows: every
    page is held by somebody, every entry of the buffers names a page or its place."""

    def __init__(self, dev, seqs, width, lens, ahead=70):
        self.dev, self.seqs, self.width = dev, seqs, width
        pages = seqs * width + 8
        gen = torch.Generator().manual_seed(seqs)
        self.all = {
            "table": torch.randint(0, pages, (seqs + 2 * ahead, width), generator=gen),
            "lens": torch.randint(0, 50, (seqs + 2 * ahead,), generator=gen),
            "refs": torch.randint(1, 5, (pages + 2 * ahead,), generator=gen)}
        self.all = {k: v.int().to(dev) for k, v in self.all.items()}
        self.table = self.all["table"][ahead:ahead + seqs]
        self.lens = self.all["lens"][ahead:ahead + seqs]
        self.refs = self.all["refs"][ahead:ahead + pages]
        self.lens.copy_(ints([lens(i) for i in range(seqs)], dev))
        self.plain = Pages(self.table, self.lens, self.refs, PAGE)

    def refused(self, op, a, b, why=2):
        """The call, by name; it must be refused, by the plain form too, and change nothing."""
        plain = getattr(self.plain, op)(a, b)
        assert (plain[0] if op == "extend" else plain) == why
        was = {k: v.clone() for k, v in self.all.items()}
        call = getattr(paged, "pages_" + op)
        last = self.extend_pools if op == "extend" else (PAGE,)
        st = call(self.table, self.lens, self.refs, ints(a, self.dev), ints(b, self.dev), *last)
        assert int(st) == why
        for k, v in self.all.items():
            assert torch.equal(v, was[k]), (op, a[:4], b[:4], k)


WILD = [-1, -PAGE, -2 * PAGE + 1, -2 * PAGE, -1000, -2 ** 31 + 15, -2 ** 31, 2 ** 31 - 1]


# one launch (entries times width at most 1024), and a launch that decides and one that moves
@pytest.mark.parametrize("seqs,width", [(6, 4), (40, 70)])
def test_refused_truncates_change_nothing(dev, seqs, width):
    g = Guarded(dev, seqs, width, lambda i: (7 * i + 5) % (width * PAGE))
    many = list(range(seqs))
    for y in WILD:
        for s in (0, seqs // 2, seqs - 1, seqs, -1, 2 ** 31 - 1, -2 ** 31):
            g.refused("truncate", [s], [y])
            keep = [0] * seqs
            if 0 <= s < seqs:
                keep[s] = y
                g.refused("truncate", many, keep)
            else:
                g.refused("truncate", many + [s], keep + [y])
    g.refused("truncate", many + [3], [0] * (seqs + 1))           # one twice
    g.refused("truncate", many, [y for y in (WILD * 8)[:seqs]])


@pytest.mark.parametrize("seqs,width", [(6, 4), (40, 70)])
def test_refused_forks_change_nothing(dev, seqs, width):
    half = seqs // 2
    g = Guarded(dev, seqs, width, lambda i: 0 if i >= half else 11 * i + 1)
    kids = list(range(half, seqs))
    parents = [i % half for i in range(len(kids))]
    for x in (seqs, -1, 2 ** 31 - 1, -2 ** 31, half):
        g.refused("fork", [x] + parents[1:], kids)                # half: a child as a parent
    for y in (seqs, -1, 2 ** 31 - 1, -2 ** 31, 0, kids[-1]):
        g.refused("fork", parents, [y] + kids[1:])                # 0: not empty; the last one twice


@pytest.mark.parametrize("seqs,width", [(6, 4), (40, 70)])
def test_refused_calls_on_broken_lengths_change_nothing(dev, seqs, width):
    # lengths that no call leaves behind: negative, or past the table
    for bad in (-1, -1000, -2 ** 31, width * PAGE + 1, 2 ** 31 - 1):
        g = Guarded(dev, seqs, width, lambda i: bad if i == 2 else 0)
        if bad > 0:                                   # the plain form knows no width here
            g.plain.truncate = g.plain.fork = lambda a, b: 2
        else:
            g.plain.fork = lambda a, b: 2
        g.refused("truncate", [2, 1], [0, 0])
        g.refused("fork", [2, 2], [1, 0])
        g.refused("truncate", list(range(seqs)), [0] * seqs)


@pytest.mark.parametrize("seqs,width", [(6, 4), (40, 70)])
def test_refused_extends_change_nothing(dev, seqs, width):
    g = Guarded(dev, seqs, width, lambda i: (7 * i + 5) % (width * PAGE))
    k = torch.randn(1, g.refs.numel(), 1, PAGE, 64, device=dev).bfloat16()
    was = k.clone()
    g.extend_pools = k, k
    many = list(range(seqs))
    for c in (-1, -PAGE, -1000, -2 ** 31, 2 ** 31 - 1, width * PAGE + 1):
        g.refused("extend", [1], [c])
        g.refused("extend", many, [0] * (seqs - 1) + [c])
    for s in (seqs, -1, 2 ** 31 - 1, -2 ** 31):
        g.refused("extend", [s], [1])
        g.refused("extend", many + [s], [0] * (seqs + 1))
    g.refused("extend", many + [3], [0] * (seqs + 1))
    g.refused("extend", [0], [PAGE], 1)                           # no page is free
    assert torch.equal(k, was)


def documented_step():
    """The step of the module's documentation."""
    return textwrap.dedent(paged.__doc__.split("in ``seqs``::\n\n", 1)[1])


# what a step meets: no pages left; a sequence at the end of its row; a sequence given twice
@pytest.mark.parametrize("pages,seqs,want", [(5, [0, 1], 1), (40, [0, 1, 3], 2), (40, [1, 1], 2),
                                             (40, [0, 1], 0)])
@pytest.mark.parametrize("captured", [False, True])
def test_the_documented_step_leaves_the_cache_when_it_is_refused(dev, pages, seqs, want, captured):
    gen = torch.Generator().manual_seed(pages)
    H, Hkv, D, layers, width = 8, 2, 64, 2, 3
    k, v, table, lens, refs = paged.new_cache(layers, pages, Hkv, PAGE, D, 5, width, device=dev)
    for x in (k, v):
        x.copy_(torch.randn(x.shape, generator=gen))
    fill = ([0, 1], [32, 20]) if pages == 5 else ([0, 1, 3], [30, 20, width * PAGE])
    paged.check(paged.pages_extend(table, lens, refs, *(ints(x, dev) for x in fill), k, v))
    paged.check(paged.pages_fork(table, lens, refs, ints([1], dev), ints([4], dev), PAGE))
    norm = [torch.ones(D, device=dev).bfloat16() for _ in range(2)]
    env = dict(paged=paged, torch=torch, k=k, v=v, table=table, lens=lens, refs=refs,
               seqs=ints(seqs, dev), layers=layers, scale=D ** -0.5, q_norm=norm[0],
               k_norm=norm[1], cos=torch.ones(width * PAGE, D, device=dev),
               sin=torch.zeros(width * PAGE, D, device=dev),
               qkv=torch.randn(layers, len(seqs), (H + 2 * Hkv) * D, generator=gen).bfloat16()
               .to(dev))
    was = [x.clone() for x in (k, v, table, lens, refs)]
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            exec(documented_step(), env)
        for x, y in zip((k, v, table, lens, refs), was):
            assert torch.equal(x, y)
        graph.replay()
    else:
        exec(documented_step(), env)
    assert int(env["status"]) == want
    if want:
        assert not env["q"].any()
        for x, y in zip((k, v, table, lens, refs), was):
            assert torch.equal(x, y)
        return
    assert lens.tolist()[:2] == [31, 21]
    for i, n in zip(seqs, (30, 20)):                 # each row's values, where its token goes
        at = int(table[i, n // PAGE])
        got = v[:, at, :, n % PAGE]
        row = env["qkv"][:, seqs.index(i)].reshape(layers, H + 2 * Hkv, D)[:, H + Hkv:]
        assert torch.equal(got, row)
    assert torch.equal(was[1][:, was[2][4, 1]], v[:, table[4, 1]])     # the fork's page is its own
