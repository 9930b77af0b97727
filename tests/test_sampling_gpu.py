"""The draw of tokens on the device against its definition in float64."""
import math

import pytest
import torch

from moss_tts_lite_amd import sampling
from tests._sampling import reference

pytestmark = pytest.mark.gpu

# Two float64 evaluations of a border differ by some 2^-48 of the whole: sums of up to 2^20 weights,
# weights in whole units of 2^-42 with random roundings.  A draw nearer than this to a border may go
# either way; the seeds here have none that near, which `check` makes sure of.
NEAR = 2.0 ** -30


def logits_of(gen, rows, vocab, typ, spread=2.0, peaks=20):
    x = spread * torch.randn(rows, vocab, generator=gen)
    for r in range(rows):
        at = torch.randperm(vocab, generator=gen)[:min(peaks, vocab)]
        x[r, at] += 6 + torch.randn(len(at), generator=gen)
    return x.to(typ)


def check(dev, logits, u, **kw):
    token, logprob = sampling.sample(logits.to(dev), u.to(dev), return_logprob=True, **{
        k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32
    ref = reference(logits, u, **kw)
    for r, (tok, lp, near) in enumerate(ref):
        assert near > NEAR, (r, near)
        assert int(token[r]) == tok, (r, int(token[r]), ref[r])
        if math.isinf(lp):
            assert float(logprob[r]) == lp
        else:                              # one rounding, and that of the largest logits' distance
            assert abs(float(logprob[r]) - lp) <= 2 ** -23 * abs(lp) + 1e-9, (r, lp)
    return token


TYPES = [torch.bfloat16, torch.float16, torch.float32]
SETTINGS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_p=0.8), dict(min_p=0.05),
            dict(top_k=40, top_p=0.9), dict(top_k=300), dict(top_k=50, min_p=0.02),
            dict(top_k=700, top_p=0.95, min_p=0.001), dict(top_p=0.999), dict(temperature=0.0),
            dict(temperature=1.7, top_p=0.6), dict(temperature=0.05), dict(top_p=0.0),
            dict(min_p=1.5), dict(min_p=1.0), dict(temperature=40.0, top_p=0.99, top_k=2000)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 1025, 8193, 40001])
def test_settings(dev, vocab, typ, kw):
    gen = torch.Generator().manual_seed(vocab)
    check(dev, logits_of(gen, 4, vocab, typ), torch.rand(4, generator=gen), **kw)


@pytest.mark.parametrize("vocab", [32767, 32768, 32769, 151936, 262145, 1 << 20])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, temperature=1.5), dict(top_p=0.95),
                                dict(min_p=0.0001), dict(top_k=5000, top_p=0.9)], ids=str)
def test_large_vocabularies(dev, vocab, kw):
    gen = torch.Generator().manual_seed(vocab + 1)
    typ = TYPES[vocab % 3]
    check(dev, logits_of(gen, 2, vocab, typ), torch.rand(2, generator=gen), **kw)


# around the sizes of a list, and min-p's border without a sum
@pytest.mark.parametrize("vocab", [700, 8192, 50000, 300001])
@pytest.mark.parametrize("kw", [dict(top_k=383), dict(top_k=385, top_p=0.97), dict(top_k=511),
                                dict(top_k=513, top_p=0.99), dict(top_k=1500),
                                dict(top_k=2500, top_p=0.9, temperature=3.0),
                                dict(top_k=4097, top_p=0.98), dict(top_k=900, min_p=0.05),
                                dict(top_k=900, top_p=0.8, min_p=0.05), dict(min_p=0.3),
                                dict(min_p=1e-6, temperature=0.2), dict(min_p=0.7, temperature=60.0),
                                dict(min_p=0.999999), dict(min_p=0.2, top_p=0.6, temperature=4.0),
                                dict(min_p=0.02, temperature=2.5),
                                dict(min_p=0.02, top_p=0.8, temperature=2.5),
                                dict(min_p=0.002, top_p=0.3, temperature=2.5),
                                dict(min_p=0.0001, top_p=0.8, temperature=2.5),
                                dict(min_p=1e-40), dict(top_k=30, min_p=1e-7)], ids=str)
def test_long_lists(dev, vocab, kw):
    gen = torch.Generator().manual_seed(vocab + 3)
    for typ in TYPES:
        check(dev, logits_of(gen, 3, vocab, typ, peaks=200), torch.rand(3, generator=gen), **kw)


@pytest.mark.parametrize("vocab", [600, 33000])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_k=400), dict(top_p=0.5),
                                dict(top_p=0.25, top_k=600), dict(min_p=0.5)], ids=str)
def test_equal_logits(dev, vocab, kw):
    # the order goes by index, and borders are met exactly: whole numbers of equal weights
    for value in (0.0, -3.5, 1e4):
        x = torch.full((3, vocab), value, dtype=torch.float16)
        x[1, ::2] = -0.0 if value == 0 else value    # -0 is 0
        x[2, : vocab // 2] = float("-inf")
        u = torch.tensor([0.0, 0.499, 0.9999])
        for r in range(3):
            live = [i for i in range(vocab) if x[r, i] != float("-inf")]
            n = min(kw.get("top_k", 0) or len(live), len(live))
            p = kw.get("top_p", 1.0)
            if p < 1:                                # tokens j with j <= p n
                n = min(n, int(math.floor(p * n)) + 1)
            want = live[min(int(float(u[r]) * n), n - 1)]
            tok = sampling.sample(x[r:r + 1].to(dev), u[r:r + 1].to(dev), **kw)
            assert int(tok) == want, (value, r)


@pytest.mark.parametrize("vocab", [9000, 70001])
@pytest.mark.parametrize("spread", [1e-5, 0.02, 30.0, 1000.0])
@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.3), dict(top_p=0.97), dict(top_k=100),
                                dict(top_p=0.6, min_p=0.3), dict(min_p=0.7),
                                dict(top_p=0.9, temperature=0.3)], ids=str)
def test_spreads(dev, vocab, spread, kw):
    # nuclei of one token to nearly all, borders among thousands of tokens of one step
    gen = torch.Generator().manual_seed(int(spread * 1e5) + vocab)
    x = spread * torch.randn(3, vocab, generator=gen) + 0.3
    check(dev, x, torch.rand(3, generator=gen), **kw)
    check(dev, x.half(), torch.rand(3, generator=gen), **kw)


@pytest.mark.parametrize("vocab", [8192, 8193, 16384, 16385, 24577])
def test_draws_in_every_chunk(dev, vocab):
    gen = torch.Generator().manual_seed(vocab)
    x = torch.randn(1, vocab, generator=gen).expand(40, vocab)
    u = (torch.arange(40).float() + 0.5) / 40
    for kw in (dict(), dict(top_p=0.9), dict(top_p=0.999)):
        tok = check(dev, x, u, **kw)
        assert (tok[1:] >= tok[:-1]).all() and int(tok[-1]) > vocab - vocab // 10


def test_borders_near_zero(dev):
    """Logits near 0 lie closer than their distances to the largest can tell apart: the border's step
    holds tokens above the logit that it begins at."""
    gen = torch.Generator().manual_seed(21)
    vocab = 40000
    x = -3 + 0.03 * torch.randn(4, vocab, generator=gen)
    for r in range(4):
        at = torch.randperm(vocab, generator=gen)[:2001]
        x[r, at] = 1e-8 * torch.randn(2001, generator=gen)
        x[r, at[0]] = 12.5 + 0.0625 * r              # distances of 12.5 .. are where steps begin
    for p in (0.05, 0.085, 0.12):
        check(dev, x, torch.rand(4, generator=gen), temperature=2.5, top_p=p)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=(1 << 20) - 1), dict(top_p=1 - 2.0 ** -24)],
                         ids=str)
def test_a_tail_of_tiny_weights(dev, kw):
    """2^20 - 1 tokens of 2^-42.1 beside one of weight 1: together 2^-22.1, which u can tell apart."""
    n = 1 << 20
    x = torch.full((1, n), -29.2)
    x[0, -1] = 0.0
    w = math.exp(float(x[0, 0]))
    u = torch.tensor([2.0 ** -23])
    assert 2.0 ** -23 < (n - 1) * w - 2.0 ** -24        # also behind top-p's border
    token, logprob = sampling.sample(x.to(dev), u.to(dev), return_logprob=True, **kw)
    # each weight counts to half of 2^-43: sums up to a token, and the whole, are off by 2^-24
    assert abs((int(token) + 1) * w - 2.0 ** -23) <= 2.0 ** -24 + 2.0 ** -40
    assert abs(float(logprob) - math.log(w)) <= 2 ** -23 * 29.2 + 2.0 ** -21


def test_large_masked_rows(dev):
    inf = float("inf")
    gen = torch.Generator().manual_seed(18)
    x = logits_of(gen, 6, 30000, torch.float32)
    x[0] = -inf
    x[1, :29999] = -inf
    x[2, 100:29000] = float("nan")
    x[3, [5, 8191, 8192, 29999]] = inf
    x[4] = torch.finfo(torch.float32).min
    x[5, 10:] = -inf
    u = torch.rand(6, generator=gen)
    for kw in (dict(), dict(top_p=0.71), dict(top_k=3), dict(min_p=0.1), dict(temperature=0.0),
               dict(top_k=20000)):
        tok = check(dev, x, u, **kw)
        assert tok[:2].tolist() == [-1, 29999] and int(tok[3]) in (5, 8191, 8192, 29999)


def test_equal_logits_of_a_large_row(dev):
    # the border lies among equals, over all chunks
    vocab = 50000
    x = torch.zeros(5, vocab, dtype=torch.bfloat16)
    x[:, 7::1000] = 1.0
    u = torch.tensor([0.0, 0.23, 0.47, 0.77, 0.9999])
    for kw in (dict(top_p=0.001), dict(top_p=0.2), dict(top_p=0.83), dict(top_k=1000),
               dict(top_k=30000, top_p=0.4), dict(min_p=0.5), dict(min_p=0.3)):
        check(dev, x, u, **kw)


def test_two_levels_of_many_ties(dev):
    gen = torch.Generator().manual_seed(5)
    x = torch.randint(0, 3, (6, 5000), generator=gen).float() * 2
    for typ in TYPES:
        for kw in (dict(top_k=1000), dict(top_k=3000), dict(top_p=0.3), dict(top_p=0.93),
                   dict(min_p=0.1), dict(min_p=0.2), dict(top_k=2500, top_p=0.7)):
            check(dev, x.to(typ), torch.rand(6, generator=gen), **kw)


def test_masked_rows(dev):
    inf = float("inf")
    gen = torch.Generator().manual_seed(8)
    x = logits_of(gen, 9, 3000, torch.float32)
    x[0] = -inf                                      # nothing is left
    x[1] = float("nan")
    x[2, 1:] = -inf                                  # one token
    x[3, :2999] = -inf
    x[4, ::2] = float("nan")
    x[5, 5:2990] = -inf                              # fewer than top_k
    x[6, [17, 40]] = inf                             # infinities share
    x[7] = torch.finfo(torch.float32).min            # the type's lowest value is a number
    x[8, 100:] = torch.finfo(torch.float32).min
    u = torch.rand(9, generator=gen)
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0),
               dict(top_k=50, top_p=0.51, min_p=0.01), dict(top_k=2000)):
        tok = check(dev, x, u, **kw)
        assert tok[:4].tolist() == [-1, -1, 0, 2999]
        assert int(tok[4]) % 2 == 1 and int(tok[6]) in (17, 40)


def test_a_setting_for_each_row(dev):
    gen = torch.Generator().manual_seed(2)
    rows = 24
    x = logits_of(gen, rows, 12000, torch.bfloat16)
    pick = lambda *z: torch.tensor([z[int(i)] for i in torch.randint(0, len(z), (rows,),
                                                                    generator=gen)])
    kw = dict(temperature=pick(0.0, 0.7, 1.0, 1.5, -1.0), top_k=pick(0, 1, 20, 500, 20000, -3).int(),
              top_p=pick(1.0, 0.9, 0.3, 2.0), min_p=pick(0.0, 0.01, 0.2))
    u = torch.rand(rows, generator=gen)
    a = check(dev, x, u, **kw)
    for r in range(rows):                            # a row draws the same by itself, by numbers
        one = sampling.sample(x[r:r + 1].to(dev), u[r:r + 1].to(dev),
                              *(float(kw[n][r]) if n != "top_k" else int(kw[n][r])
                                for n in ("temperature", "top_k", "top_p", "min_p")))
        assert int(one) == int(a[r])


@pytest.mark.parametrize("vocab", [3000, 9000, 70001])
def test_a_row_draws_the_same_in_any_batch(dev, vocab):
    """Token and probability to the last bit, whether settings are numbers or tensors and whatever the
    other rows' are; borders among ties of weights that are no whole units."""
    gen = torch.Generator().manual_seed(vocab)
    rows = 40
    x = torch.randint(0, 60, (rows, vocab), generator=gen).float() / 7
    x[::4] = x[::4].round()
    x, u = x.to(dev), torch.rand(rows, generator=gen).to(dev)
    pick = lambda *z: torch.tensor([z[int(i)] for i in torch.randint(0, len(z), (rows,),
                                                                    generator=gen)]).to(dev)
    kw = dict(temperature=pick(0.3, 0.9, 1.7), top_k=pick(0, 0, 30, 480, 700, 2500).int(),
              top_p=pick(1.0, 0.9, 0.5), min_p=pick(0.0, 0.0, 0.01))
    token, logprob = sampling.sample(x, u, return_logprob=True, **kw)
    for r in range(rows):
        one = sampling.sample(x[r:r + 1], u[r:r + 1], return_logprob=True,
                              **{k: v[r].item() for k, v in kw.items()})
        assert int(one[0]) == int(token[r]) and torch.equal(one[1], logprob[r:r + 1]), r
        mixed = {k: v[r].item() if i % 2 == r % 2 else v[r:r + 1] for i, (k, v) in
                 enumerate(kw.items())}
        two = sampling.sample(x[r:r + 1], u[r:r + 1], return_logprob=True, **mixed)
        assert torch.equal(two[0], one[0]) and torch.equal(two[1], one[1]), r


@pytest.mark.parametrize("seed", range(12))
def test_mixed_settings(dev, seed):
    # every way through a row beside every other
    gen = torch.Generator().manual_seed(100 + seed)
    rows = 12
    vocab = [5300, 8192, 8193, 30000, 65537, 151936][seed % 6]
    x = logits_of(gen, rows, vocab, TYPES[seed % 3], spread=[0.3, 1.0, 2.0, 4.0][seed % 4],
                  peaks=[1, 20, 600][seed // 4])
    pick = lambda *z: torch.tensor([z[int(i)] for i in torch.randint(0, len(z), (rows,),
                                                                    generator=gen)])
    kw = dict(temperature=pick(0.3, 0.9, 1.3, 2.0, 3.0), top_k=pick(0, 0, 30, 480, 1100, 3000).int(),
              top_p=pick(1.0, 0.95, 0.8, 0.4), min_p=pick(0.0, 0.0, 1e-4, 0.004, 0.05))
    check(dev, x, torch.rand(rows, generator=gen), **kw)


def test_random_numbers_at_the_ends(dev):
    gen = torch.Generator().manual_seed(4)
    x = logits_of(gen, 1, 2000, torch.float32).expand(6, 2000)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")])
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9)):
        ref = reference(x[:2], torch.tensor([0.0, 1 - 2.0 ** -24]), **kw)
        got = sampling.sample(x.to(dev), u.to(dev), **kw).tolist()
        assert got == [ref[0][0], ref[1][0], ref[1][0], ref[1][0], ref[0][0], ref[0][0]]


def test_extreme_temperatures(dev):
    gen = torch.Generator().manual_seed(6)
    x = logits_of(gen, 3, 5000, torch.float32)
    u = torch.rand(3, generator=gen)
    for t in (1e-30, 1e-3, 1e30):
        for kw in (dict(), dict(top_k=40), dict(top_p=0.49)):
            check(dev, x, u, temperature=t, **kw)
    inf = sampling.sample(x.to(dev), u.to(dev), torch.full((3,), float("inf"), device=dev))
    assert ((inf >= 0) & (inf < 5000)).all()
    nan = sampling.sample(x.to(dev), u.to(dev), torch.full((3,), float("nan"), device=dev))
    assert torch.equal(nan.cpu(), x.argmax(-1))


def test_every_token_is_drawn_as_often_as_it_should(dev):
    # by index the draw is exact: u on a grid finds each token for its share of the grid
    x = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5, float("-inf")]])
    n = 60000
    u = (torch.arange(n).double() / n).float()
    tok = sampling.sample(x.to(dev).expand(n, 6), u.to(dev), 0.8, top_k=4)
    w = torch.exp(x[0].double() / 0.8)
    w[[2, 5]] = 0
    share = torch.bincount(tok.cpu(), minlength=6).double() / n
    assert ((share - w / w.sum()).abs() <= 2.0 / n).all()


def test_views(dev):
    gen = torch.Generator().manual_seed(7)
    x = logits_of(gen, 5, 4001, torch.bfloat16)
    u = torch.rand(5, generator=gen).to(dev)
    want = sampling.sample(x.to(dev), u, top_k=30)
    wide = torch.empty(5, 4010, dtype=torch.bfloat16, device=dev)
    wide[:, 3:4004] = x.to(dev)
    assert torch.equal(sampling.sample(wide[:, 3:4004], u, top_k=30), want)
    assert torch.equal(sampling.sample(x.to(dev).t().contiguous().t(), u, top_k=30), want)
    assert torch.equal(sampling.sample(x.to(dev).flip(0), u.flip(0), top_k=30), want.flip(0))
    assert sampling.sample(x[:0].to(dev), u[:0]).shape == (0,)


def test_past_32_bit_offsets(dev):
    rows, vocab = 4200, 1 << 19                      # 2.2e9 logits
    x = torch.full((rows, vocab), -20.0, dtype=torch.bfloat16, device=dev)
    x[:, 3] = 5.0
    x[rows - 1, 3], x[rows - 1, vocab - 1] = -20.0, 5.0
    tok = sampling.sample(x, torch.full((rows,), 0.5, device=dev), top_k=20)
    assert (tok[:-1] == 3).all() and int(tok[-1]) == vocab - 1


def test_repeats_captures_and_streams(dev):
    gen = torch.Generator().manual_seed(9)
    x = logits_of(gen, 20, 50000, torch.bfloat16).to(dev)
    u = torch.rand(20, generator=gen).to(dev)
    t = torch.linspace(0.2, 2, 20).to(dev)
    for kw in (dict(top_k=50), dict(top_p=0.97), dict(), dict(top_k=1500, top_p=0.9),
               dict(top_p=0.8, min_p=0.02)):
        want = sampling.sample(x, u, t, return_logprob=True, **kw)
        graphs = []
        torch.cuda.synchronize()
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                got = sampling.sample(x, u, t, return_logprob=True, **kw)
            graphs.append((g, got, torch.cuda.Stream()))
        for _ in range(3):
            for g, got, s in graphs:
                with torch.cuda.stream(s):
                    got[0].fill_(-5)
                    g.replay()
            again = sampling.sample(x, u, t, return_logprob=True, **kw)
            torch.cuda.synchronize()
            for a in (again, *(got for _, got, _ in graphs)):
                assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])


def test_schemas(dev):
    from moss_tts_lite_amd import ops

    x, u = torch.randn(3, 100, device=dev), torch.rand(3, device=dev)
    for name in ("sample", "sample_logprob"):
        torch.library.opcheck(ops.overload(name), (x, u, None, None, u, None, 0.7, 5),
                              test_utils=("test_schema", "test_faketensor"))
