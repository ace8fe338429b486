"""Refusals of the paged cache's and the many-sequence attentions' entry points:
every one is decided on the host, before anything is launched."""
import ctypes as C

import pytest

import g4

L = None
P = 1 << 20      # an aligned address that is never used


@pytest.fixture(scope="module", autouse=True)
def lib():
    global L
    L = g4.Lib.get().L


def msg():
    return L.g4_last_error().decode()


def test_pool_bytes():
    rows = 5 * 32 * 2
    assert L.g4_kv_pool_bytes(g4.F32, 5, 32, 2, 256) == rows * 1024
    assert L.g4_kv_pool_bytes(g4.BF16, 5, 32, 2, 64) == rows * 128
    assert L.g4_kv_pool_bytes(g4.F16, 5, 32, 2, 128) == rows * 256
    assert L.g4_kv_pool_bytes(g4.KV_Q8, 5, 32, 2, 512) == rows * 516
    # sizes past 32 bits
    assert L.g4_kv_pool_bytes(g4.BF16, 1 << 20, 64, 8, 512) == (1 << 20) * 64 * 8 * 1024
    for bad in ((g4.Q4_K, 5, 32, 2, 256), (g4.F32, 0, 32, 2, 256), (g4.F32, 5, 8, 2, 256), (g4.F32, 5, 48, 2, 256),
                (g4.F32, 5, 8192, 2, 256), (g4.F32, 5, 32, 0, 256), (g4.F32, 5, 32, 2, 96), (g4.F32, 5, 32, 2, 0),
                (g4.F32, -1, 32, 2, 256)):
        assert L.g4_kv_pool_bytes(*bad) == 0, bad


def rows_call(fn, **kw):
    a = dict(kp=P, vp=P, type=g4.BF16, n_pages=4, page=16, n_kv=2, hd=256, table=P, ts=4, k=P, v=P, stride=512, cu=P,
             lens=P, n=3, m=10)
    a.update(kw)
    return getattr(L, fn)(*a.values())


ROWS_BAD = [dict(kp=None), dict(vp=None), dict(table=None), dict(k=None), dict(v=None), dict(cu=None), dict(lens=None),
            dict(kp=P + 8), dict(vp=P + 4), dict(k=P + 4), dict(v=P + 8), dict(n_pages=0), dict(page=24), dict(n_kv=0),
            dict(hd=200), dict(ts=0), dict(ts=(1 << 26) + 1), dict(stride=508), dict(stride=514), dict(stride=-512), dict(n=0), dict(n=4097),
            dict(m=0), dict(m=-4)]


@pytest.mark.parametrize("fn", ["g4_kv_page_store", "g4_kv_page_load"])
@pytest.mark.parametrize("bad", ROWS_BAD, ids=str)
def test_rows_refused(fn, bad):
    assert rows_call(fn, **bad) == g4.G4_ERR_ARG
    assert fn in msg()


@pytest.mark.parametrize("fn", ["g4_kv_page_store", "g4_kv_page_load"])
def test_rows_type(fn):
    assert rows_call(fn, type=g4.Q6_K) == g4.G4_ERR_TYPE
    assert "unsupported cache type 14" in msg()


def decode_call(**kw):
    a = dict(q=P, qs=2048, kp=P, vp=P, type=g4.KV_Q8, n_pages=4, page=16, n_kv=2, hd=256, table=P, ts=4, lens=P, n=3,
             window=0, heads=8, scale=C.c_float(1.0), part=P, out=P, os=2048)
    a.update(kw)
    return L.g4_attn_decode_paged(*a.values())


DECODE_BAD = [dict(q=None), dict(kp=None), dict(vp=None), dict(table=None), dict(lens=None), dict(part=None), dict(out=None),
              dict(q=P + 4), dict(out=P + 8), dict(part=P + 4), dict(qs=2044), dict(qs=2050), dict(os=2040), dict(os=2049),
              dict(heads=7), dict(heads=0), dict(n_kv=0), dict(hd=192), dict(page=0), dict(n=0), dict(n=5000),
              dict(window=-1), dict(ts=-1), dict(page=4096, ts=1 << 20)]


@pytest.mark.parametrize("bad", DECODE_BAD, ids=str)
def test_decode_refused(bad):
    assert decode_call(**bad) == g4.G4_ERR_ARG
    assert "g4_attn_decode_paged" in msg()


def test_decode_type():
    assert decode_call(type=g4.Q4_K) == g4.G4_ERR_TYPE


def test_decode_part_bytes():
    assert L.g4_attn_decode_paged_part_bytes(8, 2, 256) > 0
    for bad in ((8, 3, 256), (0, 1, 256), (8, 0, 256), (8, 2, 255), (-8, 2, 256)):
        assert L.g4_attn_decode_paged_part_bytes(*bad) == 0, bad


def prompt_call(**kw):
    a = dict(q=P, qs=2048, k=P, v=P, ks=512, out=P, os=2048, type=g4.F32, cu=P, n=3, m=10, window=0, heads=8, n_kv=2,
             hd=256, scale=C.c_float(1.0), work=P)
    a.update(kw)
    return L.g4_attn_prompt_packed(*a.values())


PROMPT_BAD = [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu=None), dict(work=None), dict(q=P + 4),
              dict(k=P + 8), dict(v=P + 4), dict(out=P + 4), dict(work=P + 8), dict(qs=2044), dict(ks=511), dict(os=2047),
              dict(type=g4.BF16, qs=2052), dict(type=g4.F16, ks=516), dict(n=0), dict(n=4097), dict(m=0), dict(window=-5),
              dict(heads=5), dict(heads=0), dict(n_kv=0), dict(hd=320)]


@pytest.mark.parametrize("bad", PROMPT_BAD, ids=str)
def test_prompt_refused(bad):
    assert prompt_call(**bad) == g4.G4_ERR_ARG
    assert "g4_attn_prompt_packed" in msg()


def test_prompt_type():
    for t in (g4.KV_Q8, g4.Q6_K, 99):
        assert prompt_call(type=t) == g4.G4_ERR_TYPE
    assert L.g4_attn_prompt_packed_work_bytes(g4.KV_Q8, 3, 10, 2, 256) == 0
    assert L.g4_attn_prompt_packed_work_bytes(g4.BF16, 3, 10, 2, 256) > 0


@pytest.mark.parametrize("fn", ["g4_kv_page_store", "g4_kv_page_load"])
@pytest.mark.parametrize("m", [(1 << 28), (1 << 31) - 1])
def test_rows_past_a_launch(fn, m):
    # a workgroup of 256 threads for every 16 rows: 2^32 threads
    assert rows_call(fn, m=m) == g4.G4_ERR_ARG
    assert fn in msg() and "launch" in msg()


@pytest.mark.parametrize("kw", [dict(m=(1 << 31) - 1), dict(m=1 << 30, type=g4.F16),
                                dict(n=4096, heads=65535, n_kv=65535, hd=64, qs=65535 * 64, ks=65535 * 64, os=65535 * 64),
                                dict(m=1 << 20, heads=65535, n_kv=1, hd=64, qs=65535 * 64, ks=64, os=65535 * 64, type=g4.BF16)],
                         ids=str)
def test_prompt_past_a_launch(kw):
    assert prompt_call(**kw) == g4.G4_ERR_ARG
    assert "g4_attn_prompt_packed" in msg() and "launch" in msg()


@pytest.mark.parametrize("pool", [(g4.F32, (1 << 31) - 1, 4096, 65535, 512), (g4.F32, 1 << 28, 4096, 8192, 512),
                                  (g4.F32, 1 << 30, 4096, 4096, 512), (g4.KV_Q8, (1 << 31) - 1, 4096, 65535, 512),
                                  (g4.BF16, 1 << 30, 4096, 4096, 512)], ids=str)
def test_pools_past_an_address(pool):
    """sizes that 64 bits do not hold are no pool, and not the size of what is left of them"""
    assert pool[1] * pool[2] * pool[3] * pool[4] * (1 if pool[0] == g4.KV_Q8 else 2) >= 1 << 63
    assert L.g4_kv_pool_bytes(*pool) == 0
    kind, pages, page, n_kv, hd = pool
    for fn in ("g4_kv_page_store", "g4_kv_page_load"):
        assert rows_call(fn, type=kind, n_pages=pages, page=page, n_kv=n_kv, hd=hd, stride=1 << 30) == g4.G4_ERR_ARG
        assert "bad pool" in msg()
    assert decode_call(type=kind, n_pages=pages, page=page, n_kv=n_kv, hd=hd, heads=n_kv) == g4.G4_ERR_ARG
    assert "bad pool" in msg()
