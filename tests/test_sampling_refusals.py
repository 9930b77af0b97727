"""What the draw of tokens refuses, before a device is touched, and its definition on the CPU."""
import ctypes

import pytest
import torch

from moss_tts_lite_amd import _native as N
from moss_tts_lite_amd import sampling
from tests._sampling import draw

FAKE = 0x10000


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def call(logits=FAKE, ld=1000, rows=2, vocab=1000, typ=N.T_F32, u=FAKE, token=FAKE, settings=True,
         ws=None, nbytes=0):
    s = ctypes.byref(N.SampleSettings(temperature_all=1.0, top_p_all=1.0)) if settings else None
    return N.load().mtl_sample(logits, ld, rows, vocab, typ, u, s, token, None, ws, nbytes, None)


def test_c_refusals():
    for kw, want in ((dict(rows=-1), N.MTL_ERR_INVALID_ARG), (dict(vocab=0), N.MTL_ERR_INVALID_ARG),
                     (dict(ld=-1), N.MTL_ERR_INVALID_ARG), (dict(settings=False), N.MTL_ERR_INVALID_ARG),
                     (dict(logits=None), N.MTL_ERR_INVALID_ARG), (dict(u=None), N.MTL_ERR_INVALID_ARG),
                     (dict(token=None), N.MTL_ERR_INVALID_ARG), (dict(typ=N.T_E4M3), N.MTL_ERR_UNSUPPORTED),
                     (dict(vocab=(1 << 20) + 1), N.MTL_ERR_SHAPE), (dict(rows=65536), N.MTL_ERR_SHAPE),
                     (dict(logits=FAKE + 2), N.MTL_ERR_ALIGN),
                     (dict(logits=FAKE + 1, typ=N.T_BF16), N.MTL_ERR_ALIGN), (dict(rows=0), N.MTL_OK)):
        assert call(**kw) == want, kw


def test_workspace():
    bytes_of = N.load().mtl_sample_workspace_bytes
    for kw in (dict(), dict(top_p_all=0.9), dict(top_k_all=50), dict(top_k=FAKE)):
        s = N.SampleSettings(**{**dict(temperature_all=1.0, top_p_all=1.0), **kw})
        assert bytes_of(2, 8192, N.T_F32, ctypes.byref(s)) == 0     # one launch does it
        need = bytes_of(2, 9000, N.T_F32, ctypes.byref(s))
        assert need > 0

        def run(ws, nbytes):
            return N.load().mtl_sample(FAKE, 9000, 2, 9000, N.T_F32, FAKE, ctypes.byref(s), FAKE,
                                       None, ws, nbytes, None)

        assert run(FAKE, need - 1) == N.MTL_ERR_WORKSPACE and run(None, need) == N.MTL_ERR_WORKSPACE
        assert run(FAKE + 8, need) == N.MTL_ERR_ALIGN
    assert bytes_of(2, 9000, N.T_F32, None) == 0 and bytes_of(0, 9000, N.T_F32, ctypes.byref(s)) == 0


@pytest.mark.parametrize("kw,what", [
    (dict(logits=meta(1000)), "rows, vocab"), (dict(logits=meta(3, 0)), "2\\^20"),
    (dict(logits=meta(3, (1 << 20) + 1)), "2\\^20"), (dict(logits=meta(65536, 8), u=meta(65536)), "rows"),
    (dict(logits=meta(3, 9, dtype=torch.float64)), "float32, bfloat16"),
    (dict(u=meta(4)), "u must"), (dict(u=meta(3, dtype=torch.float64)), "u must"),
    (dict(u=meta(3, 1)), "u must"), (dict(u=meta(6)[::2]), "u must"),
    (dict(temperature=meta(4)), "temperature must"), (dict(temperature=meta(3, dtype=torch.float64)), "temperature must"),
    (dict(top_k=meta(3)), "top_k must"), (dict(top_k=meta(3, dtype=torch.int64)), "top_k must"),
    (dict(top_p=meta(1)), "top_p must"), (dict(min_p=meta(3, 1)), "min_p must"),
    (dict(temperature=float("nan")), "finite"), (dict(temperature=float("inf")), "finite"),
    (dict(top_p=float("nan")), "numbers"), (dict(u=torch.rand(3)), "device"),
    (dict(min_p=torch.zeros(3)), "device"),
])
def test_operator_refusals(kw, what):
    with pytest.raises(RuntimeError, match=what):
        sampling.sample(**{**dict(logits=meta(3, 1000), u=meta(3)), **kw})


def test_shapes_and_host_tensors():
    assert sampling.sample(meta(3, 9), meta(3), meta(3)).dtype == torch.int64
    tok, lp = sampling.sample(meta(3, 9, dtype=torch.bfloat16), meta(3), return_logprob=True)
    assert tok.shape == lp.shape == (3,) and lp.dtype == torch.float32
    with pytest.raises(NotImplementedError):
        sampling.sample(torch.randn(2, 9), torch.rand(2))


def test_the_definition_itself():
    # the plain form that the device is compared with, on a row whose answers are known
    import math

    x = [0.0, math.log(4), math.log(2), math.log(1), float("nan"), math.log(2)]
    assert draw(x, 0.0)[0] == 0                              # weights 1 4 2 1 - 2 of 10
    for u, tok in ((0.05, 0), (0.2, 1), (0.55, 2), (0.75, 3), (0.85, 5), (0.999, 5)):
        assert draw(x, u)[0] == tok
    assert draw(x, 0.99, top_k=2)[0] == 2                    # 1 and 2 (of equals the lower index)
    assert abs(draw(x, 0.99, top_k=2)[1] - math.log(1 / 3)) < 1e-12
    assert [draw(x, u, top_p=0.45)[0] for u in (0.6, 0.7)] == [1, 2]     # 4, then 2 at index 2
    assert draw(x, 0.9, top_p=0.39)[0] == 1
    assert [draw(x, u, min_p=0.5)[0] for u in (0.0, 0.6, 0.9)] == [1, 2, 5]
    assert draw(x, 0.9, temperature=0)[0] == 1 and draw(x, 0.9, min_p=2)[0] == 1
    assert draw([float("-inf")] * 3, 0.5)[0] == -1
    assert draw([1.0, float("inf"), 2.0], 0.99)[0] == 1
