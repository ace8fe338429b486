"""GPU parity of the attention of one token over the paged cache where its work
is split over workgroups and the pieces are joined (main.c:1909-1950 of the reference for one of them)."""
import numpy as np
import pytest

import paged_np as pn
from test_gpu_paged import Cache, run_decode, within

pytestmark = pytest.mark.gpu

WIDE = 80    # further table entries: more positions than a workgroup takes whole


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


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
