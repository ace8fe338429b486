"""GPU parity of the attention of one token over the paged cache where its work
is split over workgroups and the pieces are joined, by whole heads from 256
heads of sequences on (main.c:1909-1950 of the reference for one of them)."""
import numpy as np
import pytest

import paged_np as pn
import test_gpu_paged as base
from test_gpu_paged import Cache, NAN, rows, run_decode, same, within

pytestmark = pytest.mark.gpu

WIDE = 80    # further table entries: more positions than a workgroup takes whole


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


def check(lib, seed, kind, hd, n_heads, n_kv, page, lens, window=0, scale=None, gain=3.0, joined=None):
    """as base.check_decode, with a wide table; joined: whether the pieces of whole heads are joined (else of 64 dims)"""
    if joined is not None:
        assert (n_heads * len(lens) >= 256) == joined
    assert window == 0 or window > 512
    rng = np.random.default_rng(seed)
    scale = hd ** -0.5 if scale is None else scale
    c = Cache(lib, rng, kind, hd, n_kv, page, lens, extra=WIDE)
    assert c.table.shape[1] * page > 512
    k, v = rows(rng, sum(lens), n_kv, hd), rows(rng, sum(lens), n_kv, hd)
    c.store(k, v, list(lens), lens)
    q = rows(rng, len(lens), n_heads, hd) * np.float32(gain)
    got = run_decode(lib, c, q, lens, n_heads, window, scale)
    at, hk, hv = pn.starts(lens), pn.held(k, kind, hd), pn.held(v, kind, hd)
    for s, t in enumerate(lens):
        o = got[s].reshape(n_heads, hd)
        if t == 0:
            assert (o == 0).all(), s
            continue
        r = slice(at[s], at[s + 1])
        want, bound = pn.attention(q[s].reshape(1, n_heads, hd), hk[r].reshape(t, n_kv, hd), hv[r].reshape(t, n_kv, hd),
                                   [max(0, t - window) if window else 0], scale)
        within(np.abs(o - want[0]), bound[0], (s, t))


def ragged(seed, n, top):
    rng = np.random.default_rng(seed)
    return [0, 1, 33] + [int(x) for x in np.exp(rng.uniform(0, np.log(top), n - 4))] + [top]


@pytest.mark.parametrize("kind", pn.TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_whole_heads(lib, kind, hd):
    """40 ragged sequences, 80 items; the same under a window"""
    lens = ragged(600 + hd, 40, 1700)
    check(lib, 600, kind, hd, 8, 2, 16, lens, joined=True)
    check(lib, 601, kind, hd, 8, 2, 16, lens, window=700, joined=True)


@pytest.mark.parametrize("n_heads,n_kv", [(20, 1), (40, 1), (40, 2), (8, 8)])
@pytest.mark.parametrize("kind,hd", [(pn.BF16, 128), (pn.Q8, 256), (pn.F32, 512)])
def test_heads(lib, kind, hd, n_heads, n_kv):
    """more q heads on a kv head than a workgroup takes at once, and one on each"""
    check(lib, 610 + n_heads, kind, hd, n_heads, n_kv, 32, ragged(610, 34, 900), joined=True)


@pytest.mark.parametrize("kind,hd", [(pn.F16, 256), (pn.F32, 128), (pn.Q8, 512)])
def test_few_items(lib, kind, hd):
    """whole heads joined in few items, one sequence's (no lead units) among them, and parts of 64 dims in many"""
    check(lib, 623, kind, hd, 288, 2, 16, [2100], joined=True)
    check(lib, 620, kind, hd, 16, 1, 16, ragged(620, 20, 2500), joined=True)
    check(lib, 621, kind, hd, 3, 1, 16, ragged(621, 70, 700), joined=False)
    check(lib, 622, kind, hd, 2, 2, 16, ragged(622, 90, 700), joined=False)


@pytest.mark.parametrize("kind,hd", [(pn.F32, 256), (pn.BF16, 512), (pn.Q8, 128)])
def test_pages_outside(lib, kind, hd):
    """a page outside the pool, a length past the table or below zero: NaN in that sequence's rows and nowhere else"""
    rng = np.random.default_rng(630)
    lens = np.array(ragged(630, 40, 1500), np.int32)
    c = Cache(lib, rng, kind, hd, 2, 16, lens, extra=WIDE)
    k = rows(rng, sum(lens), 2, hd)
    c.store(k, -k, list(lens), lens)
    q = rows(rng, 40, 8, hd)
    a = run_decode(lib, c, q, lens, 8, 0, 0.1)
    assert np.isfinite(a).all()
    bad = [39, 20]
    c.table[39, 50] = c.pages
    c.table[20, 0] = -1
    c.dtable = base.dbuf(lib, c.table)
    got = run_decode(lib, c, q, lens, 8, 0, 0.1)
    assert np.isnan(got[bad]).all() and same(np.delete(got, bad, 0), np.delete(a, bad, 0))
    # lengths change which workgroup takes what: the others' values stay within rounding
    lens2 = lens.copy()
    lens2[5], lens2[7] = c.table.shape[1] * 16 + 1, -2
    got = run_decode(lib, c, q, lens2, 8, 0, 0.1)
    bad += [5, 7]
    assert np.isnan(got[bad]).all()
    at, hk, hv = pn.starts(lens), pn.held(k, kind, hd), pn.held(-k, kind, hd)
    for s in range(40):
        if s not in bad and lens[s]:
            r, t = slice(at[s], at[s + 1]), lens[s]
            want, bound = pn.attention(q[s].reshape(1, 8, hd), hk[r].reshape(t, 2, hd), hv[r].reshape(t, 2, hd), [0], 0.1)
            for x in (a, got):
                within(np.abs(x[s].reshape(8, hd) - want[0]), bound[0], s)
    # what is not finite: the heads that see it and no others
    k2 = k.copy()
    k2[pn.starts(lens)[39] + 900, 3] = NAN
    c2 = Cache(lib, np.random.default_rng(630), kind, hd, 2, 16, lens, extra=WIDE)
    c2.store(k2, -k2, list(lens), lens)
    got = run_decode(lib, c2, q, lens, 8, 0, 0.1)
    assert np.isnan(got[39, :4 * hd]).all()
    a[39, :4 * hd] = got[39, :4 * hd]
    assert same(got, a)


@pytest.mark.parametrize("kind", [pn.F32, pn.BF16, pn.Q8])
@pytest.mark.parametrize("hd", [64, 512])
@pytest.mark.parametrize("lens,top,extra,step", [([160, 1, 90], 120, 0, 128), ([500, 300], 119, 0, 256),
                                                 ([1500] * 40, 117, WIDE, 128)], ids=["one", "whole", "split"])
def test_values_at_the_limit(lib, kind, hd, lens, top, extra, step):
    """V so large that the keys together stay just below fp32's largest number, under scores that rise by 2^7.9 from one
    of a wave's tiles to the next"""
    rng = np.random.default_rng(640)
    n_heads, n_kv, m = 8, 2, sum(lens)
    assert max(lens) * 2.0 ** top < float(np.finfo(np.float32).max) < max(lens) * 2.0 ** (top + 1)
    c = Cache(lib, rng, kind, hd, n_kv, 16, lens, extra=extra)
    k = np.zeros((m, n_kv, hd), np.float32)
    for a, t in zip(pn.starts(lens), lens):
        for i in range(t):
            k[a + i, :, :i // step] = 1
    k = k.reshape(m, -1)
    v = np.full((m, n_kv * hd), 2.0 ** top, np.float32) * rng.choice(np.array([1, -1], np.float32), n_kv * hd)
    q = np.zeros((len(lens), n_heads, hd), np.float32)
    q[:, :, :16] = 5.46875
    c.store(k, v, lens, lens)
    got = run_decode(lib, c, q.reshape(len(lens), -1), lens, n_heads, 0, 1.0)
    at, hk, hv = pn.starts(lens), pn.held(k, kind, hd), pn.held(v, kind, hd)
    for s, t in enumerate(lens):
        r = slice(at[s], at[s + 1])
        want, bound = pn.attention(q[s][None], hk[r].reshape(t, n_kv, hd), hv[r].reshape(t, n_kv, hd), [0], 1.0)
        within(np.abs(got[s].reshape(n_heads, hd) - want[0]), bound[0], (s, t))
