"""Refusals of the attention of chunks over the paged cache: every one is
decided on the host, before anything is launched."""
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


def call(**kw):
    a = dict(q=P, qs=2048, q_type=g4.BF16, kp=P, vp=P, type=g4.BF16, n_pages=4, page=16, n_kv=2, hd=256, table=P, ts=4, cu=P, lens=P,
             n=3, m=10, window=0, heads=8, scale=C.c_float(1.0), part=P, out=P, os=2048)
    a.update(kw)
    return L.g4_attn_chunk_paged(*a.values())


@pytest.mark.parametrize("bad", [dict(q=None), dict(kp=None), dict(vp=None), dict(table=None), dict(cu=None), dict(lens=None),
                                 dict(part=None), dict(out=None), dict(q=P + 4), dict(out=P + 8), dict(part=P + 4), dict(kp=P + 8),
                                 dict(qs=2044), dict(qs=2040), dict(os=2040), dict(os=2052), dict(q_type=g4.F32, os=2050),
                                 dict(heads=7), dict(heads=0), dict(heads=-8), dict(n_kv=0), dict(hd=192), dict(page=0), dict(n=0),
                                 dict(n=5000), dict(m=0), dict(m=-3), dict(window=-1), dict(ts=-1), dict(page=4096, ts=1 << 20),
                                 dict(heads=65538, qs=1 << 26, os=1 << 26)], ids=str)
def test_refused(bad):
    assert call(**bad) == g4.G4_ERR_ARG
    assert "g4_attn_chunk_paged" in msg()


@pytest.mark.parametrize("q,c", [(g4.F16, g4.BF16), (g4.BF16, g4.F16), (g4.F16, g4.F32), (g4.BF16, g4.F32), (g4.F16, g4.KV_Q8),
                                 (g4.KV_Q8, g4.KV_Q8), (g4.Q4_K, g4.F32), (g4.F32, g4.Q6_K)])
def test_types(q, c):
    assert call(q_type=q, type=c) == g4.G4_ERR_TYPE
    assert "g4_attn_chunk_paged" in msg()


def test_part_bytes():
    for hd in (64, 128, 256, 512):
        one = L.g4_attn_chunk_paged_part_bytes(1, 8, 2, hd)
        many = L.g4_attn_chunk_paged_part_bytes(5000, 8, 2, hd)
        assert 0 < one <= many
    for bad in ((0, 8, 2, 256), (-1, 8, 2, 256), (5, 8, 3, 256), (5, 0, 1, 256), (5, 8, 0, 256), (5, 8, 2, 255), (5, -8, 2, 256)):
        assert L.g4_attn_chunk_paged_part_bytes(*bad) == 0, bad
