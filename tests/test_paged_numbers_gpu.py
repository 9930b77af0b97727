"""Paged attention on the device against closed forms that allow nothing but the output's rounding
and float32 sums: small weights beside a dominant one, and rows whose place shows in the output."""
import math

import pytest
import torch

from moss_tts_lite_amd import paged
from tests._paged import TYPES
from tests._paged_numbers import beside, closed_form, coded_case, heads_of, room, sink_case

pytestmark = pytest.mark.gpu

KINDS = [("bf16", "bf16", 128), ("f16", "f16", 64), ("f16", "f16", 128), ("bf16", "e4m3", 64),
         ("f16", "e4m3", 128)]


def check(args, want, typ, n, drop, dev):
    a = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in args.items()}
    out, lse = (x.cpu() for x in paged.paged_attention(**a, return_lse=True))
    far = beside(out, want[0], room(n, typ, drop))
    assert not far.any(), (far.nonzero()[:4].tolist(), out[far][:4], want[0][far][:4])
    some = want[1] != float("-inf")
    assert torch.equal(lse != float("-inf"), some)
    if some.any():
        # sums of n terms, a score's and the logarithm's roundings
        tol = n * 2.0 ** -24 + (drop + 20) * 2.0 ** -22
        assert float((lse.double() - want[1])[some].abs().max()) < tol


@pytest.mark.parametrize("typ,kv,D", KINDS)
@pytest.mark.parametrize("c", [1.0, 6.0, 9.5])
@pytest.mark.parametrize("wide", [False, True])
def test_small_weights_beside_a_dominant_one(dev, typ, kv, D, c, wide):
    args, want = sink_case([300, 2, 0, 257, 470], 16, 2, D, 16, typ, kv, c, width=64 * wide)
    check(args, want, typ, 470, 1.875 * c, dev)


def test_small_weights_of_many_positions_in_a_wave(dev):
    # 512 kv heads: a workgroup takes all positions of its head, a wave every fourth tile; the
    # table names one page again and again
    heads, D, page, width = 512, 64, 256, 64
    n = width * page
    k = torch.zeros(2, heads, page, D)
    k[0, :, 0, 0] = 1
    v = (128 * (1 + torch.arange(D) % 8 / 8)).expand(2, heads, page, D).clone()
    v[0, :, 0] = 0
    table = torch.ones(1, width, dtype=torch.int32)
    table[0, 0] = 0
    q = heads_of(1, heads, D, "f16")
    few = torch.zeros(n, D, dtype=torch.float64)
    few[0, 0] = 1
    vals = v[1, 0, :1].double().repeat(n, 1)
    vals[0] = 0
    for c in (6.0, 8.8):
        out, lse = closed_form(q[:, :8], [few], [vals], c)
        want = out.repeat(1, heads // 8, 1), lse.repeat(1, heads // 8)
        args = dict(q=q, k_pages=k.half(), v_pages=v.half(), table=table,
                    lens=torch.tensor([n], dtype=torch.int32), scale=c)
        check(args, want, "f16", n, 1.875 * c, dev)


@pytest.mark.parametrize("typ,kv,D", KINDS)
@pytest.mark.parametrize("code", ["position", "tile"])
@pytest.mark.parametrize("lens", [[5000], [9001, 17], [3000, 1, 0, 2047, 4097], [700] * 33,
                                  [1, 31, 32, 33, 127, 128, 129, 500]])
def test_every_row_is_in_its_place(dev, typ, kv, D, code, lens):
    args, want = coded_case(lens, 8, 2, D, 32, typ, kv, code, seed=len(lens))
    check(args, want, typ, max(lens), 4.0, dev)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,Hkv", [(28, 4), (40, 2), (12, 12)])
def test_every_row_is_in_its_place_pages_and_heads(dev, page, H, Hkv):
    for lens in ([2500, 60, 1111], [90, 0, 256]):
        args, want = coded_case(lens, H, Hkv, 128, page, "bf16", "bf16", "position", seed=page)
        check(args, want, "bf16", max(lens), 4.0, dev)


def test_every_row_of_a_long_sequence_is_in_its_place(dev):
    for code in ("position", "tile"):
        args, want = coded_case([60001, 300, 20000], 4, 1, 64, 64, "f16", "f16", code)
        check(args, want, "f16", 60001, 4.0, dev)


@pytest.mark.parametrize("typ,kv,D", [("bf16", "bf16", 64), ("f16", "e4m3", 64)])
def test_a_hundred_million_positions(dev, typ, kv, D):
    # the same page all along: the softmax of one page, and its sum 2^19 times
    page, width = 256, 1 << 19
    args, want = coded_case([page], 2, 1, D, page, typ, kv, "position", c=4.0)
    long = dict(args, table=args["table"][:, :1].expand(1, width).contiguous(),
                lens=torch.tensor([page * width], dtype=torch.int32))
    # 512 workgroups of 4 waves: a wave takes 2^11 tiles in turn, 8 positions of each to a lane, so
    # the sums have 2^14 terms in turn and those of the join
    check(long, (want[0], want[1] + math.log(width)), typ, 1 << 14, 8.0, dev)


# ------------------------------------------------------------------------------ stored e4m3 values
def stored(x, scale):
    """x / scale as it is to be stored: one division in float32, limited, to nearest even."""
    return (x.float() / scale).clamp(-448, 448).to(torch.float8_e4m3fn)


SCALES = [1.0, 0.05, 3e-5, 2.0 ** -100, 1e-37, 2.0 ** -126, 5e-39, 2e-39, 1e-40, 2.0 ** -149, 0.0,
          1e20, 2.0 ** 100, 1e37, 3e38, float("inf"), -0.3]


@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_e4m3_values_are_divided_with_one_rounding(dev, typ):
    # a kv head a scale, subnormal and very large ones among them
    heads, D, rows = len(SCALES), 64, 64
    gen = torch.Generator().manual_seed(3)
    scale = torch.tensor(SCALES)
    x = torch.randn(rows, heads, D, generator=gen) * 3
    x = x * torch.where(scale.isfinite() & (scale != 0), scale.abs(), 1.0)[None, :, None] * 30
    x = x.to(TYPES[typ])
    x[0, :, :12] = torch.tensor([0.0, -0.0, 1.0, -1.0, float("inf"), float("-inf"), float("nan"),
                                 1e-7, 6e4, 0.5, 2.0 ** -14, -2.0 ** -24]).to(TYPES[typ])
    qkv = torch.cat([torch.zeros(rows, 1, D), x.float(), x.float().flip(0)], 1).to(TYPES[typ])
    k, v = (torch.zeros(rows, heads, 16, D, dtype=torch.float8_e4m3fn, device=dev)
            for _ in range(2))
    table = torch.arange(rows, dtype=torch.int32, device=dev)[:, None]
    paged.paged_write(qkv.reshape(rows, -1).to(dev), k, v, table,
                      torch.full((rows,), 5, device=dev), k_scale=scale.to(dev),
                      v_scale=scale.to(dev))
    for got, want in ((k, stored(x, scale[:, None])), (v, stored(x.flip(0), scale[:, None]))):
        got, want = got[:, :, 5].cpu().float(), want.float()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(), want.nan_to_num())
