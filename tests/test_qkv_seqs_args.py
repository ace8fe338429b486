"""Refusals of the packed rows' norms and rotation, as rows and into the paged
cache: every one is decided on the host, before anything is launched."""
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


def post(**kw):
    a = dict(q=P, qs=2048, qw=P, heads=8, k=P, v=P, ks=512, kw=P, n_kv=2, hd=256, qo=2 * P, qos=2048, ko=2 * P, vo=2 * P, kos=512,
             type=g4.BF16, tab=P, tab_rows=100, n_rot=256, eps=C.c_float(1e-6), cu=P, lens=P, n=3, m=10)
    a.update(kw)
    return L.g4_qkv_post_seqs(*a.values())


COMMON = [dict(qw=None), dict(qo=None), dict(v=None), dict(kw=None), dict(tab=None), dict(cu=None), dict(lens=None), dict(q=P + 4),
          dict(qw=P + 8), dict(qo=2 * P + 4), dict(k=P + 8), dict(v=P + 4), dict(kw=P + 4), dict(tab=P + 4), dict(qs=2046),
          dict(qs=2044), dict(qos=2044), dict(qos=2052), dict(ks=508), dict(ks=514), dict(heads=0), dict(heads=-1),
          dict(heads=65536, qs=1 << 25, qos=1 << 25), dict(n_kv=0), dict(n_kv=-2), dict(hd=96), dict(hd=0), dict(tab_rows=0),
          dict(tab_rows=-5), dict(n_rot=0), dict(n_rot=255), dict(n_rot=258), dict(n_rot=-2), dict(n=0), dict(n=4097), dict(m=0),
          dict(m=-1), dict(m=(1 << 31) - 1)]


@pytest.mark.parametrize("bad", COMMON + [dict(ko=None), dict(vo=None), dict(ko=2 * P + 8), dict(kos=508), dict(kos=516),
                                          dict(q=None, k=None), dict(qo=P), dict(ko=P), dict(type=g4.F32, qo=P, qos=2056),
                                          dict(type=g4.F32, vo=P, kos=520)], ids=str)
def test_post_refused(bad):
    assert post(**bad) == g4.G4_ERR_ARG
    assert "g4_qkv_post_seqs" in msg()


def test_post_type():
    for t in (g4.KV_Q8, g4.Q6_K, 99):
        assert post(type=t) == g4.G4_ERR_TYPE
        assert "unsupported row type" in msg()


def append(**kw):
    a = dict(kp=P, vp=P, type=g4.KV_Q8, n_pages=4, page=16, n_kv=2, hd=256, table=P, ts=4, k=P, v=P, ks=512, kw=P, q=P, qs=2048,
             qw=P, heads=8, qo=2 * P, qos=2048, q_type=g4.F16, tab=P, tab_rows=100, n_rot=256, eps=C.c_float(1e-6), cu=P, lens=P, n=3, m=10)
    a.update(kw)
    return L.g4_kv_page_append(*a.values())


@pytest.mark.parametrize("bad", COMMON + [dict(kp=None), dict(vp=P + 4), dict(table=None), dict(k=None), dict(n_pages=0),
                                          dict(page=48), dict(ts=0), dict(ts=(1 << 26) + 1), dict(qo=P),
                                          dict(n_kv=40000, ks=40000 * 256)], ids=str)
def test_append_refused(bad):
    assert append(**bad) == g4.G4_ERR_ARG
    assert "g4_kv_page_append" in msg()


def test_append_type():
    assert append(type=g4.Q4_K) == g4.G4_ERR_TYPE and "cache type" in msg()
    assert append(q_type=g4.KV_Q8) == g4.G4_ERR_TYPE and "q rows" in msg()


def test_more_than_a_launch_takes():
    """blocks of rows times heads are workgroups of one launch of at most 2^32 threads"""
    for m in (1 << 25, 1 << 30):
        assert post(m=m) == g4.G4_ERR_ARG and "one launch" in msg()
        assert append(m=m) == g4.G4_ERR_ARG and "one launch" in msg()
