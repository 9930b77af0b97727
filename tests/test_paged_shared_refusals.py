"""What attention with a shared prefix refuses, before a device is touched."""
import ctypes

import pytest
import torch

from moss_tts_lite_amd import _native as N
from moss_tts_lite_amd import paged
from tests.test_paged_refusals import (FAKE, POOL_ERRORS, TABLE_ERRORS, attend_args, i32, meta, pool,
                                       table)


def call(p, t, q=FAKE, ldq=4096, ldh=128, lens=FAKE, groups=FAKE, shared=FAKE, n=1, heads=32,
         typ=N.T_BF16, out=FAKE, ws=None, nbytes=0):
    return N.load().mtl_paged_attention_shared(q, ldq, ldh, ctypes.byref(p), ctypes.byref(t), lens,
                                               groups, shared, n, heads, typ, ctypes.c_float(1), out,
                                               None, ws, nbytes, None)


@pytest.mark.parametrize("kw,expect", POOL_ERRORS)
def test_pool_refusals(kw, expect):
    assert call(pool(**kw), table()) == expect


@pytest.mark.parametrize("kw,expect", TABLE_ERRORS)
def test_table_refusals(kw, expect):
    assert call(pool(), table(**kw)) == expect


def test_c_refusals():
    for kw, want in ((dict(heads=12), N.MTL_ERR_SHAPE), (dict(heads=0), N.MTL_ERR_SHAPE),
                     (dict(n=-1), N.MTL_ERR_SHAPE), (dict(n=65536), N.MTL_ERR_SHAPE),
                     (dict(typ=N.T_E4M3), N.MTL_ERR_UNSUPPORTED), (dict(q=None), N.MTL_ERR_INVALID_ARG),
                     (dict(lens=None), N.MTL_ERR_INVALID_ARG), (dict(out=None), N.MTL_ERR_INVALID_ARG),
                     (dict(groups=None), N.MTL_ERR_INVALID_ARG),
                     (dict(shared=None), N.MTL_ERR_INVALID_ARG), (dict(q=FAKE + 2), N.MTL_ERR_ALIGN),
                     (dict(ldq=4100), N.MTL_ERR_ALIGN), (dict(ldh=132), N.MTL_ERR_ALIGN)):
        assert call(pool(), table(), **kw) == want, kw
    assert call(pool(), table(seqs=0, table=None)) == N.MTL_OK
    need = N.load().mtl_paged_attention_shared_workspace_bytes(2, 1, 32, 8, 128, 1 << 16, 16)
    assert need > 0
    wide = table(width=1 << 16, ld=1 << 16)
    assert call(pool(), wide, ws=FAKE, nbytes=need - 1) == N.MTL_ERR_WORKSPACE
    assert call(pool(), wide, ws=None, nbytes=need) == N.MTL_ERR_WORKSPACE
    assert call(pool(), wide, ws=FAKE + 8, nbytes=need) == N.MTL_ERR_ALIGN


def test_limits():
    assert call(pool(), table(seqs=65536)) == N.MTL_ERR_SHAPE
    assert call(pool(), table(width=(1 << 26) + 1, ld=1 << 27)) == N.MTL_ERR_SHAPE
    assert call(pool(), table(seqs=65535, width=1 << 20, ld=1 << 20)) == N.MTL_ERR_SHAPE
    bytes_of = N.load().mtl_paged_attention_shared_workspace_bytes
    assert bytes_of(0, 1, 32, 8, 128, 4, 16) == 0 and bytes_of(2, 1, 33, 8, 128, 4, 16) == 0


def args(**kw):
    return attend_args(**{**dict(groups=i32(2), shared=i32(1)), **kw})


@pytest.mark.parametrize("kw,what", [
    (dict(groups=i32(3)), "one more than shared"), (dict(shared=i32(2)), "one more than shared"),
    (dict(groups=i32(2, 1)), "1-D"), (dict(groups=meta(2, dtype=torch.int64)), "int32"),
    (dict(shared=meta(1, dtype=torch.int64)), "int32"),
    (dict(groups=i32(65537 + 1), shared=i32(65537)), "groups"),
    (dict(groups=torch.zeros(2, dtype=torch.int32)), "device"),
    (dict(q=meta(2, 12, 128)), "multiple"), (dict(lens=i32(3)), "number of sequences"),
    (dict(q=meta(2048, 32768, 128), table=i32(2048, 4), lens=i32(2048)), "too many"),
    (dict(q=meta(60000, 32, 128), table=i32(60000, 1 << 20), lens=i32(60000)), "too many"),
])
def test_operator_refusals(kw, what):
    with pytest.raises(RuntimeError, match=what):
        paged.paged_attention_shared(**args(**kw))


def test_operator_shapes():
    out, lse = paged.paged_attention_shared(**args(), return_lse=True)
    assert out.shape == (2, 32, 128) and lse.shape == (2, 32) and lse.dtype == torch.float32
    assert paged.paged_attention_shared(**args(groups=i32(1), shared=i32(0))).shape == (2, 32, 128)


def test_every_call_the_operator_takes_fits_the_c_entry():
    # the operator's limit is inside the launch's
    import random

    rng = random.Random(1)
    for _ in range(3000):
        kv, w = rng.choice([1, 2, 8, 100]), rng.choice([1, 3, 16, 17, 64, 200])
        b, n = rng.randint(1, 65535), rng.randint(0, 65535)
        width, page = int(2 ** rng.uniform(0, 26)), rng.choice([16, 64])
        if kv * w > 65535 or width > (1 << 30) // page:
            continue
        ok = b * kv * w < 1 << 26 and (b * (-(-w // 16) + 2) + n) * (width * page // 128 + 2) < 1 << 27
        need = N.load().mtl_paged_attention_shared_workspace_bytes(b, n, kv * w, kv, 128, width, page)
        assert need > 0 or not ok, (kv, w, b, n, width, page)
