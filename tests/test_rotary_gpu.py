"""Norms and rotation of queries and keys on the device against float64."""
import math

import pytest
import torch

from moss_tts_lite_amd import paged, rotary
from tests._paged import HALF_STEP, TYPES

pytestmark = pytest.mark.gpu

SMALLEST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}    # half a step of subnormal numbers


def rotary64(x, positions, freqs, norm, eps, interleaved, amplitude):
    """(value, size of the terms) in float64 on the host, pair by pair."""
    x = x.detach().cpu().double()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.cpu().double()
    y, mag = x.clone(), x.abs()
    half = len(freqs)
    a = positions.cpu().double()[:, None] * freqs.cpu().double()[None]
    for t in range(half):
        i, j = (2 * t, 2 * t + 1) if interleaved else (t, t + half)
        c, s = (f(a[:, t])[:, None] * amplitude for f in (torch.cos, torch.sin))
        y[..., i] = x[..., i] * c - x[..., j] * s
        y[..., j] = x[..., j] * c + x[..., i] * s
        mag[..., i] = mag[..., j] = abs(amplitude) * (x[..., i].abs() + x[..., j].abs())
    pad = (positions.cpu() < 0)[:, None, None]
    return y.masked_fill(pad, 0), mag


def check(got, x, positions, freqs, norm, eps, interleaved, amplitude):
    ref, mag = rotary64(x, positions, freqs, norm, eps, interleaved, amplitude)
    # one rounding, and in float32: the sum of squares (head_dim / 64 + 14 roundings, halved), its
    # root, three products (2^-20 together), cosine and sine (2^-21 of a part's rounding and the
    # function's)
    tol = HALF_STEP[got.dtype] * ref.abs() + 2.0 ** -19 * mag + SMALLEST[got.dtype]
    worst = ((got.cpu().double() - ref).abs() - tol).max()
    assert float(worst) <= 0, float(worst)


def case(dev, rows, H, Hkv, D, turned, typ="bf16", norm=True, far=5000, seed=0, pad=0):
    gen = torch.Generator().manual_seed(seed)
    t = TYPES[typ]
    buf = torch.randn(rows, (H + 2 * Hkv) * D + pad, generator=gen).to(t).to(dev)
    qkv = buf[:, :(H + 2 * Hkv) * D]
    q = qkv[:, :H * D].unflatten(1, (H, D))
    k = qkv[:, H * D:(H + Hkv) * D].unflatten(1, (Hkv, D))
    pos = torch.randint(0, far, (rows,), generator=gen)
    w = [(1 + torch.randn(D, generator=gen) / 8).to(t).to(dev) if norm else None for _ in range(2)]
    freqs = rotary.rotary_freqs(turned, 1e6, device=dev)
    return buf, dict(q=q, k=k, positions=pos.to(dev), freqs=freqs, q_norm=w[0], k_norm=w[1])


def run_case(a, eps=1e-6, interleaved=False, amplitude=1.0):
    q, k = rotary.qk_rotary(**a, eps=eps, interleaved=interleaved, amplitude=amplitude)
    assert q.is_contiguous() and q.shape == a["q"].shape and k.shape == a["k"].shape
    for got, x, w in ((q, "q", "q_norm"), (k, "k", "k_norm")):
        check(got, a[x], a["positions"], a["freqs"], a[w], eps, interleaved, amplitude)
    return q, k


@pytest.mark.parametrize("D,turned", [(8, 8), (16, 2), (64, 64), (64, 32), (80, 80), (80, 40),
                                      (80, 6), (96, 48), (128, 128), (128, 64), (128, 16),
                                      (128, 0), (128, 126), (192, 192), (256, 256), (256, 100),
                                      (264, 264), (512, 512)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("typ,norm", [("bf16", True), ("f16", False)])
def test_head_sizes_and_parts(dev, D, turned, interleaved, typ, norm):
    _, a = case(dev, 5, 6, 2, D, turned, typ, norm, seed=D + turned)
    run_case(a, interleaved=interleaved, amplitude=1.25)


@pytest.mark.parametrize("rows,H,Hkv", [(1, 1, 1), (1, 32, 8), (3, 40, 2), (17, 7, 1), (512, 4, 4),
                                        (513, 4, 4), (1100, 32, 8)])
def test_rows_and_heads(dev, rows, H, Hkv):
    _, a = case(dev, rows, H, Hkv, 128, 128, seed=rows, pad=24)
    run_case(a)


@pytest.mark.parametrize("first", [0, 1 << 20, (1 << 31) - 3, (1 << 40) + 12345, (1 << 53) - 9])
def test_far_positions(dev, first):
    # the definition in whole numbers: frequencies that are 2^-j of a turn in float64
    _, a = case(dev, 8, 4, 1, 64, 64, norm=False, seed=1)
    a["positions"] = torch.arange(first, first + 8, device=dev)
    j = torch.arange(32).double() + 1
    a["freqs"] = (2 * math.pi * 2.0 ** -j).to(dev)
    q, _ = rotary.qk_rotary(**a)
    # position times 2^-j turns, reduced exactly; 2 pi itself is off by 2^-53 of itself in float64,
    # which position 2^53 makes a part of a turn: there the float64 number's own angle counts
    x = a["q"].cpu().double()
    two_pi = 2 * math.pi
    off = 2.4492935982947064e-16                     # 2 pi - fl(2 pi)
    for i, p in enumerate(range(first, first + 8)):
        for t in range(32):
            whole = (p % (1 << (t + 1))) / (1 << (t + 1))
            ang = two_pi * whole - p * 2.0 ** -(t + 1) * off
            c, s = math.cos(ang), math.sin(ang)
            u, v = x[i, :, t], x[i, :, t + 32]
            for got, ref in ((q[i, :, t], u * c - v * s), (q[i, :, t + 32], v * c + u * s)):
                tol = HALF_STEP[q.dtype] * ref.abs() + 2.0 ** -19 * (u.abs() + v.abs())
                assert ((got.cpu().double() - ref).abs() <= tol).all(), (p, t)


def test_padding_and_in_place(dev):
    for interleaved in (False, True):
        buf, a = case(dev, 9, 4, 2, 80, 40, seed=4, pad=16)
        a["positions"][[0, 4, 8]] = torch.tensor([-1, -(1 << 40), -7], device=dev)
        q, k = run_case(a, interleaved=interleaved)
        before = buf.clone()
        rotary.qk_rotary_(**a, interleaved=interleaved)
        pads = a["positions"] < 0
        cols = torch.zeros(buf.shape[1], dtype=torch.bool, device=dev)
        cols[:6 * 80] = True
        assert torch.equal(buf[:, ~cols], before[:, ~cols]) and torch.equal(buf[pads], before[pads])
        assert torch.equal(a["q"][~pads], q[~pads]) and torch.equal(a["k"][~pads], k[~pads])
        assert not q[pads].any() and not k[pads].any()


def test_views_and_special_values(dev):
    gen = torch.Generator().manual_seed(3)
    D = 64
    q = torch.randn(D, 6, 5, generator=gen).bfloat16().to(dev).permute(2, 1, 0)   # no adjacent dims
    k = torch.randn(1, 1, D, generator=gen).bfloat16().to(dev).expand(5, 3, D)    # broadcast
    pos = torch.arange(5, device=dev)
    freqs = rotary.rotary_freqs(D, device=dev)
    run_case(dict(q=q, k=k, positions=pos, freqs=freqs, q_norm=None, k_norm=None))
    odd = torch.randn(5 * 6 * D + 1, generator=gen).bfloat16().to(dev)[1:].view(5, 6, D)
    run_case(dict(q=odd, k=k, positions=pos, freqs=freqs, q_norm=odd[0, 0].clone(), k_norm=None))
    # zeros stay zeros under the norm, an infinity or NaN stays in its head
    z = torch.zeros(2, 3, D, device=dev, dtype=torch.float16)
    z[0, 1, 5], z[1, 2, 0] = float("inf"), float("nan")
    w = torch.ones(D, device=dev, dtype=torch.float16)
    got, _ = rotary.qk_rotary(z, z, torch.arange(2, device=dev), freqs, w, w)
    bad = got.isnan().any(-1)
    assert bad.tolist() == [[False, True, False], [False, False, True]]
    assert not got[~bad].any()


def test_no_rows_and_no_heads(dev):
    f = rotary.rotary_freqs(64, device=dev)
    e = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev)
    p = torch.empty(0, dtype=torch.int64, device=dev)
    assert rotary.qk_rotary(e, e, p, f)[0].shape == (0, 4, 64)
    rotary.qk_rotary_(e, e[:, :2], p, f)
    q, none = torch.randn(3, 4, 64, device=dev).bfloat16(), e.new_empty(3, 0, 64)
    got, k = rotary.qk_rotary(q, none, torch.arange(3, device=dev), f)
    check(got, q, torch.arange(3), f, None, 1e-6, False, 1.0)
    assert k.shape == (3, 0, 64)


def test_past_32_bit_offsets(dev):
    rows, H, D = 70000, 240, 128                     # 2.15e9 elements of q
    q = torch.empty(rows, H, D, dtype=torch.bfloat16, device=dev)
    pick = torch.tensor([0, 1, 34953, rows - 1], device=dev)
    q[pick] = torch.randn(4, H, D, device=dev).bfloat16()
    pos = torch.full((rows,), -1, device=dev)
    pos[pick] = pick
    f = rotary.rotary_freqs(D, device=dev)
    before = q[pick].clone()
    k = q.new_empty(rows, 0, D)
    rotary.qk_rotary_(q, k, pos, f)
    check(q[pick], before, pick, f, None, 1e-6, False, 1.0)


def test_captured_and_on_another_stream(dev):
    _, a = case(dev, 40, 8, 2, 128, 64, seed=9)
    want = rotary.qk_rotary(**a)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        got = rotary.qk_rotary(**a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for x in got:
            x.fill_(1)
        g.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            other = rotary.qk_rotary(**a)
        s.synchronize()
        for x, y, z in zip(got, other, want):
            assert torch.equal(x, z) and torch.equal(y, z)
    a["positions"].add_(17)                          # the graph reads where its tensors are now
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], rotary.qk_rotary(**a)[0])


def test_as_the_paged_write_rotates(dev):
    # whole heads, half against half, out of a float32 table: the same rows into the same pages
    H, Hkv, D, n = 8, 2, 128, 33
    buf, a = case(dev, n, H, Hkv, D, D, seed=6)
    a["positions"] = torch.arange(n, device=dev)
    ang = torch.outer(a["positions"].double(), a["freqs"])
    cos, sin = (torch.cat([f(ang)] * 2, -1).float() for f in (torch.cos, torch.sin))
    pools = [[torch.zeros(5, Hkv, 16, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
             for _ in range(2)]
    table = torch.arange(5, dtype=torch.int32, device=dev)[None]
    seqs = torch.zeros(n, dtype=torch.int32, device=dev)
    q0 = paged.paged_write(buf, *pools[0], table, a["positions"], seqs, a["q_norm"], a["k_norm"],
                           cos, sin)
    rotary.qk_rotary_(**a)
    q1 = paged.paged_write(buf, *pools[1], table, a["positions"], seqs)
    for x, y in ((q0, q1), (pools[0][0], pools[1][0])):
        # a float32 angle part or table entry apart: at a tie the next step
        assert ((x.double() - y.double()).abs() <= 2 ** -7 * y.double().abs() + 2.0 ** -18).all()
        assert (x != y).float().mean() < 0.01
    assert torch.equal(pools[0][1], pools[1][1])


def test_schemas(dev):
    from moss_tts_lite_amd import ops

    _, a = case(dev, 3, 4, 2, 64, 32, seed=1)
    for name in ("qk_rotary", "qk_rotary_"):
        torch.library.opcheck(ops.overload(name), tuple(a.values()),
                              test_utils=("test_schema", "test_faketensor"))
