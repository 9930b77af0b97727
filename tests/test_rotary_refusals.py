"""What the rotation of queries and keys refuses, before a device is touched, and the frequencies."""
import ctypes
import math

import pytest
import torch

from moss_tts_lite_amd import _native as N
from moss_tts_lite_amd import rotary

FAKE = 0x10000


def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def heads(**kw):
    f = dict(x=FAKE, x_row=1024, x_head=128, out=FAKE + (1 << 20), out_row=1024, out_head=128,
             norm=None, heads=8)
    f.update(kw)
    return N.RotaryHeads(**f)


def call(q, k=None, rows=2, dim=128, pos=FAKE, freqs=FAKE, turned=128, typ=N.T_BF16):
    k = k if k is not None else heads(heads=0)
    return N.load().mtl_qk_rotary(ctypes.byref(q), ctypes.byref(k), rows, dim, pos, freqs, turned,
                                  0, ctypes.c_float(1), ctypes.c_float(1e-6), typ, None)


def test_c_refusals():
    for kw, want in ((dict(rows=-1), N.MTL_ERR_INVALID_ARG), (dict(pos=None), N.MTL_ERR_INVALID_ARG),
                     (dict(freqs=None), N.MTL_ERR_INVALID_ARG), (dict(dim=0), N.MTL_ERR_SHAPE),
                     (dict(dim=132), N.MTL_ERR_SHAPE), (dict(dim=520), N.MTL_ERR_SHAPE),
                     (dict(turned=130), N.MTL_ERR_SHAPE), (dict(turned=3), N.MTL_ERR_SHAPE),
                     (dict(turned=-2), N.MTL_ERR_SHAPE), (dict(rows=(1 << 25) + 1), N.MTL_ERR_SHAPE),
                     (dict(typ=N.T_E4M3), N.MTL_ERR_UNSUPPORTED), (dict(rows=0), N.MTL_OK)):
        assert call(heads(), **kw) == want, kw
    for kw, want in ((dict(x=None), N.MTL_ERR_INVALID_ARG), (dict(out=None), N.MTL_ERR_INVALID_ARG),
                     (dict(heads=-1), N.MTL_ERR_INVALID_ARG), (dict(x=FAKE + 2), N.MTL_ERR_ALIGN),
                     (dict(out_row=1020), N.MTL_ERR_ALIGN), (dict(norm=FAKE + 8), N.MTL_ERR_ALIGN),
                     (dict(out=FAKE, out_row=2048), N.MTL_ERR_INVALID_ARG),
                     (dict(heads=65536), N.MTL_ERR_SHAPE)):
        assert call(heads(**kw)) == want, kw
        assert call(heads(heads=0), heads(**kw)) == want, kw
    assert call(heads(heads=0)) == N.MTL_OK


def args(**kw):
    a = dict(q=meta(5, 8, 128), k=meta(5, 2, 128), positions=meta(5, dtype=torch.int64),
             freqs=meta(64, dtype=torch.float64))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(q=meta(5, 8, 128, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(k=meta(5, 2, 128, dtype=torch.float16)), "one type"), (dict(q=meta(5, 1024)), "heads"),
    (dict(k=meta(4, 2, 128)), "same rows"), (dict(k=meta(5, 2, 64)), "same rows"),
    (dict(q=meta(5, 8, 132), k=meta(5, 2, 132)), "multiple of 8"),
    (dict(q=meta(5, 8, 520), k=meta(5, 2, 520)), "multiple of 8"),
    (dict(q=meta(5, 65536, 128)), "65535 heads"), (dict(positions=meta(5, dtype=torch.int32)), "int64"),
    (dict(positions=meta(4, dtype=torch.int64)), "positions"),
    (dict(freqs=meta(64, dtype=torch.float32)), "float64"),
    (dict(freqs=meta(65, dtype=torch.float64)), "turned at most"),
    (dict(freqs=meta(128, dtype=torch.float64)[::2]), "contiguous float64"),
    (dict(q_norm=meta(64)), "norm"), (dict(k_norm=meta(128, dtype=torch.float32)), "norm"),
    (dict(positions=torch.zeros(5, dtype=torch.int64)), "device"),
])
def test_operator_refusals(kw, what):
    for f in (rotary.qk_rotary, rotary.qk_rotary_):
        with pytest.raises(RuntimeError, match=what):
            f(**args(**kw))


def test_in_place_refusals():
    qkv = meta(5, 12 * 128)
    q, k = qkv[:, :1024].unflatten(1, (8, 128)), qkv[:, 1024:1280].unflatten(1, (2, 128))
    rotary.qk_rotary_(**args(q=q, k=k))
    rotary.qk_rotary_(**args(q=k, k=qkv[:, 1280:].unflatten(1, (2, 128))))
    one = meta(12, 5, 128).transpose(0, 1)                   # heads before rows
    rotary.qk_rotary_(**args(q=one[:, :8], k=one[:, 8:]))
    for kw, what in ((dict(q=q, k=qkv[:, 896:1152].unflatten(1, (2, 128))), "share memory"),
                     (dict(q=q, k=q), "share memory"),
                     (dict(q=meta(1, 8, 128).expand(5, 8, 128)), "overlap"),
                     (dict(k=meta(5, 1, 128).expand(5, 2, 128)), "overlap"),
                     (dict(q=meta(5, 128, 8).transpose(1, 2)), "in place"),
                     (dict(q=meta(5, 8, 132)[..., :128]), "in place")):
        with pytest.raises(RuntimeError, match=what):
            rotary.qk_rotary_(**args(**kw))


def test_shapes_and_host_tensors():
    q, k = rotary.qk_rotary(**args(q=meta(5, 128, 8).transpose(1, 2)))
    assert q.shape == (5, 8, 128) and k.shape == (5, 2, 128) and q.is_contiguous()
    with pytest.raises(NotImplementedError):
        rotary.qk_rotary(torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, 1, 64).bfloat16(),
                         torch.zeros(1, dtype=torch.int64), torch.zeros(32, dtype=torch.float64))


def test_frequencies():
    f = rotary.rotary_freqs(128, 1e6, device="cpu")
    assert f.dtype == torch.float64 and len(f) == 64 and f[0] == 1
    assert torch.allclose(f, torch.tensor([1e6 ** (-2 * t / 128) for t in range(64)],
                                          dtype=torch.float64), rtol=1e-14)
    assert torch.equal(rotary.rotary_freqs(128, 1e6, 4.0, device="cpu"), f / 4)
    g = rotary.rotary_freqs(128, 1e6, 8.0, original=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32])
    assert torch.equal(g[turns <= 1], f[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (g[mid] < f[mid]).all() and (g[mid] > f[mid] / 8).all()
    assert (g[1:] < g[:-1]).all()
    assert rotary.rotary_freqs(0, device="cpu").numel() == 0
    assert rotary.rotary_amplitude(1.0) == 1 and rotary.rotary_amplitude(0.5) == 1
    assert abs(rotary.rotary_amplitude(8.0) - 1.2079441541679836) < 1e-12
    for kw in (dict(turned=3), dict(turned=-2), dict(turned=8, base=0.0), dict(turned=8, factor=0.0),
               dict(turned=8, factor=2.0, original=0),
               dict(turned=8, factor=2.0, original=64, slow=4.0, fast=4.0)):
        with pytest.raises(RuntimeError):
            rotary.rotary_freqs(**kw, device="cpu")


@pytest.mark.parametrize("turned,base,factor,original,slow,fast,a,b", [
    (128, 1e6, 4.0, 32768, 1.0, 32.0, 23, 40), (64, 1e4, 8.0, 4096, 1.0, 32.0, 10, 23),
    (128, 5e5, 2.0, 8192, 2.0, 16.0, 21, 32), (96, 1e7, 40.0, 2048, 1.0, 64.0, 4, 18)])
def test_frequencies_that_fall_from_dim_to_dim(turned, base, factor, original, slow, fast, a, b):
    """What rope type "yarn" means: from the dim of `fast` turns, rounded down, to that of `slow`
    turns, rounded up, in equal steps."""
    turns = [original * base ** (-2 * t / turned) / (2 * math.pi) for t in (a, a + 1, b - 1, b)]
    assert turns[0] >= fast > turns[1] and turns[2] > slow >= turns[3]
    f = rotary.rotary_freqs(turned, base, factor, original, slow, fast, "cpu")
    for t in range(turned // 2):
        g = 1.0 if t <= a else 0.0 if t >= b else (b - t) / (b - a)
        want = base ** (-2 * t / turned) * (g + (1 - g) / factor)
        assert abs(float(f[t]) - want) <= 1e-12 * want, t


def test_frequencies_that_fall_with_the_turns():
    # wavelengths of original / 4 and shorter keep theirs, of original and longer are divided
    f = rotary.rotary_freqs(128, 5e5, device="cpu")
    g = rotary.rotary_freqs(128, 5e5, 8.0, 8192, slow=1.0, fast=4.0, device="cpu", ramp="turns")
    for t in range(64):
        n = 8192 * float(f[t]) / (2 * math.pi)
        keep = min(max((n - 1) / 3, 0), 1)
        want = float(f[t]) * (keep + (1 - keep) / 8)
        assert abs(float(g[t]) - want) <= 1e-12 * want, t
    # some of the values that such a checkpoint's program has, in float32
    for t, part in ((28, 1.0), (29, 0.8281684), (32, 0.3711222), (34, 0.1902107), (35, 0.125)):
        assert abs(float(g[t] / f[t]) - part) <= 3e-7


def test_frequencies_of_short_contexts():
    f = rotary.rotary_freqs(64, 1e4, device="cpu")
    # no dim makes a turn; none makes 32 (dim 0 begins the fall); all make 32
    assert torch.equal(rotary.rotary_freqs(64, 1e4, 4.0, 6, device="cpu"), f / 4)
    g = rotary.rotary_freqs(64, 1e4, 4.0, 100, device="cpu")
    assert g[0] == f[0] and (g[1:] < f[1:]).all() and torch.equal(g[10:], f[10:] / 4)
    assert torch.equal(rotary.rotary_freqs(64, 1e4, 4.0, 1 << 30, device="cpu"), f)
    assert torch.equal(rotary.rotary_freqs(64, 1e4, 4.0, 6, device="cpu", ramp="turns"), f / 4)
    assert rotary.rotary_freqs(0, 1e4, 4.0, 100, device="cpu").numel() == 0
    for kw in (dict(ramp="dim"), dict(base=1.0), dict(base=0.5), dict(slow=0.0)):
        with pytest.raises(RuntimeError):
            rotary.rotary_freqs(**{**dict(turned=64, factor=4.0, original=100, device="cpu"), **kw})


def test_infinite_settings_of_frequencies():
    inf = float("inf")
    for kw in (dict(original=inf), dict(fast=inf), dict(base=inf), dict(slow=float("nan"))):
        with pytest.raises(RuntimeError):
            rotary.rotary_freqs(**{**dict(turned=64, factor=4.0, original=100, device="cpu"), **kw})
