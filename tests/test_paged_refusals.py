"""The paged cache's entry points refuse what their documentation rules out, before a device is
touched: the C entries by status, the torch operators (on meta tensors, which run the same
checks) by RuntimeError, and host tensors (CPU only)."""
import ctypes

import pytest
import torch

from moss_tts_lite_amd import _native as N
from moss_tts_lite_amd import paged

FAKE = 0x10000          # never dereferenced: every call below fails validation or has no work


@pytest.fixture(scope="module")
def lib():
    return N.load()


def pool(**kw):
    f = dict(k=FAKE, v=FAKE, pages=4, k_page=8 * 16 * 128, k_head=16 * 128, k_token=128,
             v_page=8 * 16 * 128, v_head=16 * 128, v_token=128, kv_heads=8, page_size=16,
             head_dim=128, type=N.T_BF16, k_scale=None, v_scale=None)
    f.update(kw)
    return N.PagePool(**f)


def table(**kw):
    f = dict(table=FAKE, ld=4, width=4, seqs=2)
    f.update(kw)
    return N.PageTable(**f)


POOL_ERRORS = [
    (dict(k=None), N.MTL_ERR_INVALID_ARG), (dict(pages=0), N.MTL_ERR_INVALID_ARG),
    (dict(pages=1 << 31), N.MTL_ERR_INVALID_ARG), (dict(kv_heads=0), N.MTL_ERR_INVALID_ARG),
    (dict(head_dim=96), N.MTL_ERR_SHAPE), (dict(page_size=24), N.MTL_ERR_SHAPE),
    (dict(page_size=512), N.MTL_ERR_SHAPE), (dict(type=N.T_F16), N.MTL_ERR_UNSUPPORTED),
    (dict(type=7), N.MTL_ERR_UNSUPPORTED), (dict(k_scale=FAKE), N.MTL_ERR_UNSUPPORTED),
    (dict(k_token=132), N.MTL_ERR_ALIGN), (dict(v_page=-8), N.MTL_ERR_ALIGN),
    (dict(v=FAKE + 8), N.MTL_ERR_ALIGN), (dict(type=N.T_E4M3, k_head=8), N.MTL_ERR_ALIGN),
]
TABLE_ERRORS = [(dict(table=None), N.MTL_ERR_INVALID_ARG), (dict(ld=3), N.MTL_ERR_INVALID_ARG),
                (dict(seqs=-1), N.MTL_ERR_INVALID_ARG), (dict(width=-1), N.MTL_ERR_INVALID_ARG)]


def attention(lib, p, t, q=FAKE, ldq=4096, ldh=128, lens=FAKE, heads=32, typ=N.T_BF16, out=FAKE,
              ws=None, nbytes=0):
    return lib.mtl_paged_attention(q, ldq, ldh, ctypes.byref(p), ctypes.byref(t), lens, heads, typ,
                                   ctypes.c_float(1), out, None, ws, nbytes, None)


def write(lib, p, t, qkv=FAKE, ldq=6144, rows=2, pos=FAKE, norms=(None, None), rope=(None, None),
          heads=32, typ=N.T_BF16, q=FAKE):
    return lib.mtl_paged_write(qkv, ldq, rows, ctypes.byref(p), ctypes.byref(t), pos, None, *norms,
                               *rope, 0, 0, ctypes.c_float(1e-6), heads, typ, q, None)


@pytest.mark.parametrize("kw,expect", POOL_ERRORS)
def test_pool_refusals(lib, kw, expect):
    assert attention(lib, pool(**kw), table()) == expect
    assert write(lib, pool(**kw), table()) == expect


@pytest.mark.parametrize("kw,expect", TABLE_ERRORS)
def test_table_refusals(lib, kw, expect):
    assert attention(lib, pool(), table(**kw)) == expect
    assert write(lib, pool(), table(**kw)) == expect


def test_attention_refusals(lib):
    ws = 1 << 30
    assert attention(lib, pool(), table(), heads=12) == N.MTL_ERR_SHAPE
    assert attention(lib, pool(), table(), heads=0) == N.MTL_ERR_SHAPE
    assert attention(lib, pool(), table(), typ=N.T_E4M3) == N.MTL_ERR_UNSUPPORTED
    assert attention(lib, pool(), table(), q=None) == N.MTL_ERR_INVALID_ARG
    assert attention(lib, pool(), table(), lens=None) == N.MTL_ERR_INVALID_ARG
    assert attention(lib, pool(), table(), q=FAKE + 2) == N.MTL_ERR_ALIGN
    assert attention(lib, pool(), table(), ldq=4100) == N.MTL_ERR_ALIGN
    assert attention(lib, pool(), table(seqs=0, table=None)) == N.MTL_OK      # nothing to do
    need = lib.mtl_paged_attention_workspace_bytes(2, 32, 8, 128, 1 << 16, 16)
    if need:
        assert attention(lib, pool(), table(width=1 << 16, ld=1 << 16), ws=FAKE,
                         nbytes=need - 1) == N.MTL_ERR_WORKSPACE
        assert attention(lib, pool(), table(width=1 << 16, ld=1 << 16), ws=None,
                         nbytes=ws) == N.MTL_ERR_WORKSPACE


def test_launch_limits(lib):
    # more threads than a launch can have: refused, not left to the launch
    p = dict(kv_heads=256, k_page=256 * 16 * 128, v_page=256 * 16 * 128)
    assert attention(lib, pool(**p), table(width=1, ld=1, seqs=65535), heads=256,
                     ldq=256 * 128) == N.MTL_ERR_SHAPE
    assert write(lib, pool(), table(), rows=1 << 24) == N.MTL_ERR_SHAPE
    assert attention(lib, pool(), table(seqs=65536)) == N.MTL_ERR_SHAPE
    assert attention(lib, pool(), table(width=(1 << 26) + 1, ld=1 << 27)) == N.MTL_ERR_SHAPE


def test_write_refusals(lib):
    assert write(lib, pool(), table(), norms=(FAKE, None)) == N.MTL_ERR_INVALID_ARG
    assert write(lib, pool(), table(), rope=(None, FAKE)) == N.MTL_ERR_INVALID_ARG
    assert write(lib, pool(), table(), rows=-1) == N.MTL_ERR_INVALID_ARG
    assert write(lib, pool(), table(), ldq=6136) == N.MTL_ERR_SHAPE
    assert write(lib, pool(), table(), ldq=6148) == N.MTL_ERR_ALIGN
    assert write(lib, pool(), table(), qkv=None) == N.MTL_ERR_INVALID_ARG
    assert write(lib, pool(), table(), rows=0, qkv=None) == N.MTL_OK


def state(**kw):
    f = dict(table=FAKE, ld=4, width=4, seqs=2, lens=FAKE, refs=FAKE, pages=8, page_size=16)
    f.update(kw)
    return N.PageState(**f)


@pytest.mark.parametrize("kw,n,expect", [
    (dict(table=None), 1, N.MTL_ERR_INVALID_ARG), (dict(lens=None), 1, N.MTL_ERR_INVALID_ARG),
    (dict(refs=None), 1, N.MTL_ERR_INVALID_ARG), (dict(ld=2), 1, N.MTL_ERR_INVALID_ARG),
    (dict(pages=-1), 1, N.MTL_ERR_INVALID_ARG), (dict(page_size=48), 1, N.MTL_ERR_SHAPE),
    (dict(page_size=0), 1, N.MTL_ERR_SHAPE), (dict(seqs=32769), 1, N.MTL_ERR_SHAPE),
    (dict(width=(1 << 20) + 1, ld=1 << 21), 1, N.MTL_ERR_SHAPE), (dict(), 1025, N.MTL_ERR_SHAPE),
    (dict(), -1, N.MTL_ERR_INVALID_ARG)])
def test_bookkeeping_refusals(lib, kw, n, expect):
    st = ctypes.byref(state(**kw))
    ws = (FAKE, 1 << 30, None)
    assert lib.mtl_pages_extend(st, FAKE, FAKE, n, FAKE, FAKE, FAKE, FAKE, *ws) == expect
    assert lib.mtl_pages_fork(st, FAKE, FAKE, n, FAKE, *ws) == expect
    assert lib.mtl_pages_truncate(st, FAKE, FAKE, n, FAKE, *ws) == expect


def test_bookkeeping_workspace_and_pointers(lib):
    st = ctypes.byref(state())
    need = lib.mtl_pages_workspace_bytes(2, 8)
    assert lib.mtl_pages_extend(st, FAKE, FAKE, 2, FAKE, FAKE, FAKE, FAKE, FAKE, need - 1,
                                None) == N.MTL_ERR_WORKSPACE
    assert lib.mtl_pages_extend(st, FAKE, FAKE, 2, FAKE, FAKE, FAKE, FAKE, FAKE + 4, need,
                                None) == N.MTL_ERR_ALIGN
    for i in range(5):                    # counts, sources, destinations, their number, status
        p = [FAKE] * 5
        p[i] = None
        assert lib.mtl_pages_extend(st, FAKE, p[0], 2, *p[1:], FAKE, need,
                                    None) == N.MTL_ERR_INVALID_ARG
    assert lib.mtl_pages_fork(st, None, FAKE, 2, FAKE, FAKE, need, None) == N.MTL_ERR_INVALID_ARG
    assert lib.mtl_pages_compact(st, FAKE, 3, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, need,
                                 None) == N.MTL_ERR_INVALID_ARG
    assert lib.mtl_pages_compact(st, FAKE, 4, FAKE, FAKE, FAKE, None, FAKE, FAKE, need,
                                 None) == N.MTL_ERR_INVALID_ARG


def test_copy_refusals(lib):
    def copy(k=FAKE, layers=2, kl=1 << 20, kp=4096, page=4096, pages=8, src=FAKE, n=2):
        return lib.mtl_pages_copy(k, FAKE, layers, kl, kl, kp, kp, page, pages, src, FAKE, n, None,
                                  None)

    assert copy(kp=2048) == N.MTL_ERR_INVALID_ARG
    assert copy(layers=-1) == N.MTL_ERR_INVALID_ARG
    assert copy(src=None) == N.MTL_ERR_INVALID_ARG
    assert copy(k=FAKE + 4) == N.MTL_ERR_ALIGN
    assert copy(kl=(1 << 20) + 8) == N.MTL_ERR_ALIGN
    assert copy(layers=65536) == N.MTL_ERR_SHAPE
    for kw in (dict(layers=0), dict(n=0), dict(pages=0), dict(page=0)):
        assert copy(**kw) == N.MTL_OK


# ------------------------------------------------------------------ torch operators (meta tensors)
def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def i32(*shape):
    return meta(*shape, dtype=torch.int32)


def attend_args(**kw):
    a = dict(q=meta(2, 32, 128), k_pages=meta(9, 8, 16, 128), v_pages=meta(9, 8, 16, 128),
             table=i32(2, 4), lens=i32(2), scale=0.1)
    a.update(kw)
    return a


E4 = torch.float8_e4m3fn


@pytest.mark.parametrize("kw,what", [
    (dict(q=meta(2, 32, 128, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(q=meta(2, 32, 128, dtype=torch.float16)), "rows' type"),
    (dict(q=meta(2, 32, 64)), "head_dim"), (dict(q=meta(2, 12, 128)), "multiple"),
    (dict(q=meta(3, 32, 128)), "number of sequences"), (dict(q=meta(2, 4096)), "sequences, heads"),
    (dict(lens=i32(3)), "number of sequences"),
    (dict(lens=meta(2, dtype=torch.int64)), "int32"),
    (dict(table=meta(2, 4, dtype=torch.int64)), "int32"), (dict(table=i32(4)), "2-D"),
    (dict(table=i32(4, 2).t()), "unit last stride"), (dict(table=i32(1, 4).expand(2, 4)), "overlap"),
    (dict(k_pages=meta(9, 8, 16, 96), v_pages=meta(9, 8, 16, 96)), "head_dim must"),
    (dict(k_pages=meta(9, 8, 24, 128), v_pages=meta(9, 8, 24, 128)), "page_size"),
    (dict(k_pages=meta(9, 8, 8, 128), v_pages=meta(9, 8, 8, 128)), "page_size"),
    (dict(v_pages=meta(8, 8, 16, 128)), "same shape"),
    (dict(v_pages=meta(9, 8, 16, 128, dtype=E4)), "same shape and type"),
    (dict(k_pages=meta(0, 8, 16, 128), v_pages=meta(0, 8, 16, 128)), "at least one page"),
    (dict(k_pages=meta(9, 8, 128, 16).transpose(2, 3)), "unit last stride"),
    (dict(k_pages=meta(9, 8, 16, 132)[..., :128]), "16 bytes"),
    (dict(k_pages=meta(2, 9, 8, 16, 128)), "kv_heads"),
    (dict(k_scale=meta(8, dtype=torch.float32)), "e4m3"),
    (dict(k_pages=meta(9, 8, 16, 128, dtype=E4), v_pages=meta(9, 8, 16, 128, dtype=E4),
          v_scale=meta(7, dtype=torch.float32)), "v_scale"),
    (dict(k_pages=meta(9, 8, 16, 128, dtype=E4), v_pages=meta(9, 8, 16, 128, dtype=E4),
          k_scale=meta(8)), "k_scale"),
    (dict(lens=torch.zeros(2, dtype=torch.int32)), "device"),
])
def test_attention_operator_refusals(kw, what):
    with pytest.raises(RuntimeError, match=what):
        paged.paged_attention(**attend_args(**kw))


def test_attention_operator_shapes():
    out = paged.paged_attention(**attend_args())
    assert out.shape == (2, 32, 128) and out.dtype == torch.bfloat16 and out.is_contiguous()
    out, lse = paged.paged_attention(**attend_args(), return_lse=True)
    assert lse.shape == (2, 32) and lse.dtype == torch.float32


def write_args(**kw):
    a = dict(qkv=meta(5, 48 * 128), k_pages=meta(9, 8, 16, 128), v_pages=meta(9, 8, 16, 128),
             table=i32(6, 4), positions=meta(5, dtype=torch.int64))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(qkv=meta(5, 16 * 128)), "columns"), (dict(qkv=meta(5, 48 * 128 + 64)), "columns"),
    (dict(qkv=meta(5, 6144, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(positions=i32(5)), "int64"), (dict(positions=meta(4, dtype=torch.int64)), "positions"),
    (dict(seqs=i32(4)), "seqs"), (dict(seqs=meta(5, dtype=torch.int64)), "int32"),
    (dict(table=i32(4, 4)), "row r is sequence r"),
    (dict(q_norm=meta(128)), "both q_norm"), (dict(q_norm=meta(128), k_norm=meta(64)), "norm"),
    (dict(q_norm=meta(128, dtype=torch.float32), k_norm=meta(128)), "norm"),
    (dict(cos=meta(64, 128)), "both cos"),
    (dict(cos=meta(64, 128), sin=meta(64, 128, dtype=torch.float32)), "cos and sin"),
    (dict(cos=meta(64, 64), sin=meta(64, 64)), "cos and sin"),
    (dict(v_scale=meta(8, dtype=torch.float32)), "e4m3"),
])
def test_write_operator_refusals(kw, what):
    with pytest.raises(RuntimeError, match=what):
        paged.paged_write(**write_args(**kw))
    assert paged.paged_write(**write_args()).shape == (5, 32, 128)


def test_pages_that_overlap_are_not_written():
    one = meta(1, 8, 16, 128).expand(9, 8, 16, 128)
    with pytest.raises(RuntimeError, match="single memory location"):
        paged.paged_write(**write_args(k_pages=one))
    with pytest.raises(RuntimeError, match="single memory location"):
        paged.paged_write(**write_args(v_pages=meta(9, 1, 16, 128).expand(9, 8, 16, 128)))
    layers = meta(1, 9, 8, 16, 128).expand(2, 9, 8, 16, 128)
    for k, v in ((layers, meta(2, 9, 8, 16, 128)), (meta(2, 9, 8, 16, 128), layers)):
        with pytest.raises(RuntimeError, match="single memory location"):
            paged.pages_copy(k, v, i32(2), i32(2))
        with pytest.raises(RuntimeError, match="single memory location"):
            paged.pages_compact(i32(6, 4), i32(9), k, v)
    assert paged.paged_attention(**attend_args(k_pages=one, v_pages=one)).shape == (2, 32, 128)


def book(**kw):
    a = dict(table=i32(6, 4), lens=i32(6), refs=i32(9))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,what", [
    (dict(table=i32(6)), "2-D"), (dict(lens=i32(5)), "lens"), (dict(refs=i32(3, 3)), "1-D"),
    (dict(refs=meta(9, dtype=torch.int64)), "int32"),
    (dict(table=i32(32769, 1), lens=i32(32769)), "at most"),
])
def test_bookkeeping_operator_refusals(kw, what):
    k = meta(2, 9, 8, 16, 128)
    two = i32(2), i32(2)
    with pytest.raises(RuntimeError, match=what):
        paged.pages_extend(**book(**kw), seqs=two[0], counts=two[1], k_pages=k, v_pages=k)
    with pytest.raises(RuntimeError, match=what):
        paged.pages_fork(**book(**kw), parents=two[0], children=two[1], page_size=16)
    with pytest.raises(RuntimeError, match=what):
        paged.pages_truncate(**book(**kw), seqs=two[0], new_lens=two[1], page_size=16)


def test_bookkeeping_operator_call_refusals():
    k = meta(2, 9, 8, 16, 128)
    for a, b, what in ((i32(2), i32(3), "same length"), (i32(1025), i32(1025), "at most"),
                       (meta(2, dtype=torch.int64), i32(2), "int32")):
        with pytest.raises(RuntimeError, match=what):
            paged.pages_extend(**book(), seqs=a, counts=b, k_pages=k, v_pages=k)
        with pytest.raises(RuntimeError, match=what):
            paged.pages_truncate(**book(), seqs=a, new_lens=b, page_size=16)
    with pytest.raises(RuntimeError, match="page_size"):
        paged.pages_fork(**book(), parents=i32(2), children=i32(2), page_size=20)
    with pytest.raises(RuntimeError, match="counts"):
        paged.pages_extend(**book(refs=i32(8)), seqs=i32(2), counts=i32(2), k_pages=k, v_pages=k)
    assert paged.pages_extend(**book(), seqs=i32(2), counts=i32(2), k_pages=k,
                              v_pages=k).shape == (1,)


@pytest.mark.parametrize("k,what", [
    (meta(9, 8, 16), "leading layers"), (meta(2, 9, 8, 16, 128, dtype=torch.float32), "e4m3fn"),
    (meta(2, 9, 8, 16, 256)[..., :128], "one block"), (meta(2, 9, 8, 32, 128)[:, :, :, :16], "block"),
])
def test_pool_block_refusals(k, what):
    with pytest.raises(RuntimeError, match=what):
        paged.pages_copy(k, k, i32(2), i32(2))
    with pytest.raises(RuntimeError, match=what):
        paged.pages_compact(i32(6, 4), i32(9), k, k)


def test_pool_block_forms():
    # transposed pages and K and V side by side in one tensor are blocks too
    k = meta(2, 9, 16, 8, 128).transpose(2, 3)
    both = meta(2, 9, 2, 8, 16, 128)
    paged.pages_copy(k, k, i32(2), i32(2))
    paged.pages_copy(both[:, :, 0], both[:, :, 1], i32(2), i32(2))
    paged.pages_copy(k[0], k[1], i32(0), i32(0))
    with pytest.raises(RuntimeError, match="same length"):
        paged.pages_copy(k, k, i32(2), i32(3))
    t, r, live = paged.pages_compact(i32(6, 4), i32(9), k, k)
    assert t.shape == (6, 4) and r.shape == (9,) and live.shape == (1,)


def test_host_tensors_are_refused():
    t = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        paged.pages_fork(t, t[:, 0], t[0], t[0], t[0], 16)


def test_check_reads_a_status():
    paged.check(torch.tensor([0]))
    for code, what in ((1, "free pages"), (2, "given twice")):
        with pytest.raises(RuntimeError, match=what):
            paged.check(torch.tensor([code]))


# ------------------------------------------------------------------ limits, checked before a device
@pytest.mark.parametrize("kv", [65536, 1 << 32, (1 << 32) + 8])
def test_more_kv_heads_than_a_launch_takes(kv):
    # 2^32 heads of stride 0 were 0 in the launch's 32 bits, and q's heads divided by that
    k = meta(9, 1, 16, 128).expand(9, kv, 16, 128)
    with pytest.raises(RuntimeError, match="65535 kv heads"):
        paged.paged_attention(**attend_args(k_pages=k, v_pages=k))
    with pytest.raises(RuntimeError, match="65535 kv heads"):
        paged.paged_write(**write_args(k_pages=k, v_pages=k))


def test_more_work_than_a_launch_takes():
    many = meta(1, 1, 128).expand(2, 65536, 128)
    with pytest.raises(RuntimeError, match="65535 heads"):
        paged.paged_attention(**attend_args(q=many))
    with pytest.raises(RuntimeError, match="65535 sequences"):
        paged.paged_attention(**attend_args(q=meta(65536, 32, 128), table=i32(65536, 4),
                                            lens=i32(65536)))
    with pytest.raises(RuntimeError, match="2\\^30 positions"):
        paged.paged_attention(**attend_args(table=i32(2, (1 << 26) + 1)))
    with pytest.raises(RuntimeError, match="rows"):
        paged.paged_write(**write_args(qkv=meta(1 << 24, 48 * 128), table=i32(1 << 24, 4),
                                       positions=meta(1 << 24, dtype=torch.int64)))
    with pytest.raises(RuntimeError, match="pages a sequence"):
        paged.pages_fork(**book(table=i32(6, (1 << 20) + 1)), parents=i32(2), children=i32(2),
                         page_size=16)
    assert paged.paged_attention(**attend_args(table=i32(2, 1 << 26))).shape == (2, 32, 128)


# ------------------------------------------------------------------ memory that two places share
def test_keys_and_values_in_the_same_memory_are_not_written():
    both = meta(2 * 9, 8, 16, 128)
    with pytest.raises(RuntimeError, match="single memory location|share memory"):
        paged.paged_write(**write_args(k_pages=both[:9], v_pages=both[:9]))
    with pytest.raises(RuntimeError, match="single memory location|share memory"):
        paged.paged_write(**write_args(k_pages=both[:9], v_pages=both[4:13]))
    with pytest.raises(RuntimeError, match="single memory location|share memory"):
        paged.pages_copy(both[:9], both[4:13], i32(2), i32(2))
    assert paged.paged_write(**write_args(k_pages=both[:9], v_pages=both[9:])).shape == (5, 32, 128)
    side = meta(9, 2, 8, 16, 128)
    q = paged.paged_write(**write_args(k_pages=side[:, 0], v_pages=side[:, 1]))
    assert q.shape == (5, 32, 128)
    assert paged.paged_attention(**attend_args(k_pages=both[:9], v_pages=both[4:13])).shape == \
        (2, 32, 128)


@pytest.mark.parametrize("strides", [(8 * 16 * 128 - 128, 16 * 128, 128, 1),       # pages meet
                                     (8 * 16 * 128, 8 * 128, 128, 1),              # heads meet
                                     (16 * 128, 16 * 128, 128, 1)])
def test_pages_that_meet_are_not_written(strides):
    k = torch.as_strided(meta(9 * 8 * 16 * 128), (9, 8, 16, 128), strides)
    with pytest.raises(RuntimeError, match="overlap"):
        paged.paged_write(**write_args(k_pages=k))
    with pytest.raises(RuntimeError, match="overlap"):
        paged.paged_write(**write_args(v_pages=k))
    # a page of 17 rows to a head, tokens first, layers inside pages: nothing meets
    for sizes, st in (((9, 8, 16, 128), (8 * 17 * 128, 17 * 128, 128, 1)),
                      ((9, 8, 16, 128), (16 * 8 * 128, 128, 8 * 128, 1)),
                      ((9, 8, 16, 128), (16 * 128, 9 * 16 * 128, 128, 1)),
                      ((9, 1, 16, 128), (16 * 128, 3, 128, 1))):
        k = torch.as_strided(meta(9 * 8 * 17 * 128), sizes, st)
        a = write_args(k_pages=k, v_pages=meta(*sizes))
        assert paged.paged_write(**a).shape == (5, 48 - 2 * sizes[1], 128)


def test_layers_that_meet_are_not_copied():
    page = 8 * 16 * 128
    k = torch.as_strided(meta(18 * page), (2, 9, 8, 16, 128), (8 * page, page, 16 * 128, 128, 1))
    with pytest.raises(RuntimeError, match="overlap"):
        paged.pages_copy(k, meta(2, 9, 8, 16, 128), i32(2), i32(2))
    inside = meta(9, 2, 8, 16, 128).transpose(0, 1)
    paged.pages_copy(inside, meta(2, 9, 8, 16, 128), i32(2), i32(2))
