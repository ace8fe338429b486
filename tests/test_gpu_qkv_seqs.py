"""Norms and rotation of packed rows (main.c:1886-1900 of the reference, which
has one sequence), as rows and straight into the paged cache, against the
formulas in 64 bits and, bit for bit, against the calls they stand for."""
import ctypes as C

import numpy as np
import pytest

import paged_np as pn
from test_gpu_paged import Cache, Stream, dbuf, filled, rows, same_bits, within

pytestmark = pytest.mark.gpu

F = C.c_float
EPS = 1e-6
NP = {pn.F32: np.float32, pn.F16: np.uint16, pn.BF16: np.uint16}


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


def table_of(rng, positions, n_rot):
    a = rng.uniform(-np.pi, np.pi, (positions, n_rot // 2))
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def plain(x, heads, hd, w, cs):
    """(y, bound) in 64 bits: rows x [rows, heads * hd], weights w (None: neither weight nor rotation), pairs cs of each row.

    The fp32 sum of squares is a product and at most 8 + 6 sums deep (2^-24 each, all terms positive); the division by hd
    is exact, eps, root and reciprocal are three roundings and halve what came before: below 7.5 + 3 for s, then w s, x (w s),
    two products and a sum: 15 halves of an ulp of the larger product's magnitude, taken as 16."""
    x = np.asarray(x, np.float64).reshape(len(x), heads, hd)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    if w is None:
        return y, 16 * 2.0 ** -24 * np.abs(y)
    y = y * np.asarray(w, np.float64)
    half = cs.shape[1]
    c, s = (np.asarray(cs[:, None, :, i], np.float64) for i in (0, 1))
    a, b = y[..., :half].copy(), y[..., hd // 2:hd // 2 + half].copy()
    mag = np.abs(y)
    y[..., :half], y[..., hd // 2:hd // 2 + half] = a * c - b * s, a * s + b * c
    mag[..., :half] = np.abs(a * c) + np.abs(b * s)
    mag[..., hd // 2:hd // 2 + half] = np.abs(a * s) + np.abs(b * c)
    return y, 16 * 2.0 ** -24 * mag


def read(buf, kind, shape):
    a = buf.to_array(NP[kind]).reshape(shape)
    return a if kind == pn.F32 else a.view(np.float16).astype(np.float32) if kind == pn.F16 else pn.bf16_back(a)


def close(got, want, bound, kind, at):
    got = got.reshape(want.shape).astype(np.float64)
    # half an ulp of the type (of its smallest normal number below that), of a value that is off by the bound already
    least = {pn.F32: 2.0 ** -150, pn.F16: 2.0 ** -25, pn.BF16: 2.0 ** -134}[kind]
    within(np.abs(got - want), bound * (1 + pn.HALF[kind]) + (pn.HALF[kind] * np.abs(want) if kind != pn.F32 else 0) + least + 1e-37, at)


def size_of(kind):
    return 4 if kind == pn.F32 else 2


class Rows:
    """q, k, v rows of ragged sequences on the device, with weights and a table"""

    def __init__(self, lib, rng, n, lens, heads, kv, hd, n_rot, pad=3, wide=8, spare=5):
        self.lib, self.n, self.lens, self.heads, self.kv, self.hd, self.n_rot = lib, n, lens, heads, kv, hd, n_rot
        self.m = sum(n) + pad
        self.x = []
        for h in (heads, kv, kv):
            r = rows(rng, self.m, 1, h * hd + wide) * np.exp(rng.standard_normal((self.m, 1))).astype(np.float32)
            r[sum(n):] = np.nan
            self.x.append(r)
        self.w = [rng.uniform(0.25, 1.75, hd).astype(np.float32) for _ in range(2)]
        self.tab = table_of(rng, max(max(lens), 1) + spare, n_rot)
        self.d = [dbuf(lib, a) for a in (*self.x, *self.w, self.tab, pn.starts(n), np.asarray(lens, np.int32))]
        self.pos = np.concatenate([np.arange(l - t, l) for t, l in zip(n, lens)] + [[]]).astype(int)

    def q_in(self):
        return self.d[0].ptr, self.x[0].shape[1], self.d[3].ptr, self.heads

    def kv_in(self):
        return self.d[1].ptr, self.d[2].ptr, self.x[1].shape[1], self.d[4].ptr

    def turn(self, tab_rows=None):
        return self.d[5].ptr, tab_rows or len(self.tab), self.n_rot, F(EPS)

    def seqs(self):
        return self.d[6].ptr, self.d[7].ptr, len(self.n), self.m

    def outs(self, kind, wide=16):
        return [filled(self.lib, self.m * (h * self.hd + wide) * size_of(kind), 0x3F) for h in (self.heads, self.kv, self.kv)]

    def post(self, kind, q=True, k=True, wide=16, tab_rows=None):
        o = self.outs(kind, wide)
        self.lib.g4_qkv_post_seqs(*(self.q_in() if q else (None, 0, None, 0)), *(self.kv_in() if k else (None, None, 0, None)),
                                  self.kv if k else 0, self.hd, o[0].ptr, self.heads * self.hd + wide, o[1].ptr, o[2].ptr,
                                  self.kv * self.hd + wide, kind, *self.turn(tab_rows), *self.seqs())
        self.lib.g4_sync()
        return o

    def want(self, i, used):
        h = self.heads if i == 0 else self.kv
        x = self.x[i][:used, :h * self.hd]
        return plain(x, h, self.hd, self.w[i] if i < 2 else None, self.tab[self.pos])


N = [5, 0, 1, 33, 16, 64, 2]
LENS = [5, 9, 40, 133, 31, 64, 1000]


@pytest.mark.parametrize("kind", [pn.F32, pn.F16, pn.BF16])
@pytest.mark.parametrize("heads,kv,hd,n_rot", [(3, 1, 64, 64), (4, 2, 64, 22), (5, 2, 128, 128), (8, 2, 256, 256),
                                               (2, 2, 256, 126), (8, 2, 512, 512), (3, 1, 512, 2)])
def test_rows(lib, kind, heads, kv, hd, n_rot):
    """ragged sequences with and without earlier positions; wide strides and padding stay as they are"""
    rng = np.random.default_rng(hd + n_rot + heads)
    r = Rows(lib, rng, N, LENS, heads, kv, hd, n_rot)
    o = r.post(kind)
    used = sum(N)
    for i, h in enumerate((heads, kv, kv)):
        raw = o[i].to_array(np.uint8).reshape(r.m, -1)
        assert (raw[used:] == 0x3F).all() and (raw[:, h * hd * size_of(kind):] == 0x3F).all()
        got = read(o[i], kind, (r.m, h * hd + 16))[:used, :h * hd]
        close(got, *r.want(i, used), kind, (i, kind, hd))


@pytest.mark.parametrize("hd,n_rot", [(256, 256), (256, 64), (512, 512)])
def test_bits_of_rows_form(lib, hd, n_rot):
    """fp32 results are g4_qkv_post_rows' with the positions' table rows gathered, bit for bit; in place too"""
    rng = np.random.default_rng(hd)
    heads, kv = 8, 2
    r = Rows(lib, rng, N, LENS, heads, kv, hd, n_rot, pad=0, wide=0)
    o = r.post(pn.F32, wide=0)
    q = dbuf(lib, r.x[0])
    ko, vo = (filled(lib, r.m * kv * hd * 4) for _ in range(2))
    tab = dbuf(lib, r.tab[r.pos])
    lib.g4_qkv_post_rows(q.ptr, r.d[3].ptr, r.d[1].ptr, r.d[2].ptr, r.d[4].ptr, ko.ptr, vo.ptr, kv * hd, tab.ptr, r.m, heads, kv,
                         hd, n_rot, F(EPS))
    lib.g4_sync()
    for a, b in zip(o, (q, ko, vo)):
        assert same_bits(a.to_array(np.float32), b.to_array(np.float32))
    lib.g4_qkv_post_seqs(*r.q_in(), *r.kv_in(), kv, hd, r.d[0].ptr, heads * hd, r.d[1].ptr, r.d[2].ptr, kv * hd, pn.F32, *r.turn(),
                         *r.seqs())
    lib.g4_sync()
    for a, b in zip(o, r.d):
        assert same_bits(a.to_array(np.float32), b.to_array(np.float32))


@pytest.mark.parametrize("hd", [64, 512])
def test_one_side_only(lib, hd):
    """q without k and v, and the other way round: the same bits, the other rows left alone"""
    rng = np.random.default_rng(hd + 1)
    r = Rows(lib, rng, N, LENS, 6, 3, hd, hd)
    both = [b.to_array(np.uint8) for b in r.post(pn.BF16)]
    q, k, v = [b.to_array(np.uint8) for b in r.post(pn.BF16, k=False)]
    assert same_bits(q, both[0]) and (k == 0x3F).all() and (v == 0x3F).all()
    q, k, v = [b.to_array(np.uint8) for b in r.post(pn.BF16, q=False)]
    assert same_bits(k, both[1]) and same_bits(v, both[2]) and (q == 0x3F).all()


def test_many_sequences(lib):
    """more sequences than a wave has lanes, most of a row or none"""
    rng = np.random.default_rng(5)
    n = [int(i) for i in rng.integers(0, 4, 333)]
    n[100] = 77
    lens = [int(t + h) for t, h in zip(n, rng.integers(0, 300, 333))]
    r = Rows(lib, rng, n, lens, 2, 1, 128, 128)
    o = r.post(pn.F32)
    for i, h in enumerate((2, 1, 1)):
        got = read(o[i], pn.F32, (r.m, h * 128 + 16))[:sum(n), :h * 128]
        close(got, *r.want(i, sum(n)), pn.F32, i)


def test_misfits_are_skipped(lib):
    """a sequence with more rows than positions, past the table, or past the rows: left as it is, the others done"""
    rng = np.random.default_rng(6)
    n, lens = [5, 7, 4, 9], [9, 6, 40, 12]
    r = Rows(lib, rng, n, lens, 2, 1, 64, 64, pad=0)
    o = r.post(pn.F32, tab_rows=20)
    got = o[0].to_array(np.uint8).reshape(r.m, -1)
    left = (got == 0x3F).all(1)
    assert list(left) == [False] * 5 + [True] * 11 + [False] * 9
    r.m = 24                                     # one less than the rows of the last sequence
    assert (r.post(pn.F32, tab_rows=20)[0].to_array(np.uint8).reshape(24, -1)[16:] == 0x3F).all()


@pytest.mark.parametrize("row", [0.0, 1e-30, 1e18, np.inf, np.nan])
def test_extremes(lib, row):
    """rows of zeros, of squares below and above fp32's, infinities and NaN: the formula in fp32, and the rows beside them
    as they would be"""
    rng = np.random.default_rng(7)
    r = Rows(lib, rng, [20], [20], 2, 1, 256, 256, pad=0, wide=0)
    want = [read(b, pn.F32, (20, -1)) for b in r.post(pn.F32, wide=0)]
    for i in range(3):
        r.x[i][7] = row
        r.d[i].write(r.x[i])
    got = [read(b, pn.F32, (20, -1)) for b in r.post(pn.F32, wide=0)]
    for i, (g, w) in enumerate(zip(got, want)):
        keep = np.arange(20) != 7
        assert same_bits(g[keep], w[keep])
        if np.isfinite(row):
            y, bound = r.want(i, 20)
            close(g[7:8], y[7:8], bound[7:8], pn.F32, (row, i))
        else:
            assert np.isnan(g[7]).all()


@pytest.mark.parametrize("kind", pn.TYPES)
@pytest.mark.parametrize("heads,kv,hd,page,q_kind", [(4, 2, 64, 16, pn.F32), (6, 1, 128, 64, pn.BF16), (8, 2, 256, 16, pn.F16),
                                                     (8, 2, 512, 32, pn.BF16), (3, 3, 256, 4096, pn.F32)])
def test_append(lib, kind, heads, kv, hd, page, q_kind):
    """the rows form to fp32 rows and g4_kv_page_store of them, bit for bit: every byte of the pools and the q rows; the
    first turns, then a token each, in codes their scales too"""
    rng = np.random.default_rng(hd + page + kind)
    n_rot = hd // 2 if heads == 6 else hd
    turns = [(N, LENS), ([1] * 7, [l + 1 for l in LENS])]
    one, two = (Cache(lib, np.random.default_rng(1), kind, hd, kv, page, [l + 1 for l in LENS]) for _ in range(2))
    for n, lens in turns:
        r = Rows(lib, rng, n, lens, heads, kv, hd, n_rot)
        qo = r.outs(q_kind)[0]
        lib.g4_kv_page_append(*one.args(), *r.kv_in(), *r.q_in(), qo.ptr, heads * hd + 16, q_kind, *r.turn(), *r.seqs())
        lib.g4_sync()
        assert same_bits(qo.to_array(np.uint8), r.post(q_kind, k=False)[0].to_array(np.uint8))
        f = r.post(pn.F32, q=False)
        lib.g4_kv_page_store(*two.args(), f[1].ptr, f[2].ptr, kv * hd + 16, r.d[6].ptr, r.d[7].ptr, len(n), r.m)
        lib.g4_sync()
        for a, b in ((one.k, two.k), (one.v, two.v)):
            assert same_bits(a.to_array(np.uint8), b.to_array(np.uint8))


def test_append_without_q_and_bad_pages(lib):
    """no q rows; pages outside the pool are dropped, sequences past the page table skipped with their q rows"""
    rng = np.random.default_rng(8)
    n, lens = [20, 3, 6], [40, 50, 6]
    c = Cache(lib, rng, pn.BF16, 128, 1, 16, [40, 32, 6], extra=0)      # sequence 1: past its table (48 positions)
    c.table[0, 1] = c.pages
    c.dtable.write(c.table)
    r = Rows(lib, rng, n, lens, 2, 1, 128, 128)
    r.lib.g4_kv_page_append(*c.args(), *r.kv_in(), None, 0, None, 0, None, 0, 0, *r.turn(), *r.seqs())
    lib.g4_sync()
    bare = [c.k.to_array(np.uint8), c.v.to_array(np.uint8)]
    for b in (c.k, c.v):
        lib.g4_memset(b.ptr, 0xFF, b.nbytes)
    qo = r.outs(pn.F32)[0]
    lib.g4_kv_page_append(*c.args(), *r.kv_in(), *r.q_in(), qo.ptr, 2 * 128 + 16, pn.F32, *r.turn(), *r.seqs())
    lib.g4_sync()
    assert same_bits(bare[0], c.k.to_array(np.uint8)) and same_bits(bare[1], c.v.to_array(np.uint8))
    left = (qo.to_array(np.uint8).reshape(r.m, -1) == 0x3F).all(1)
    assert list(left[:29]) == [False] * 20 + [True] * 3 + [False] * 6
    gk, _ = c.load([20, 0, 6], [40, 0, 6])
    bad = np.isnan(gk[:26]).all(1)
    # positions 20 .. 31 of sequence 0 lie in the bad page
    assert list(bad) == [True] * 12 + [False] * 14


def test_captured(lib):
    """a captured append follows lengths, row starts and rows through its replays"""
    rng = np.random.default_rng(9)
    heads, kv, hd, page = 4, 2, 256, 16
    with Stream(lib):
        r = Rows(lib, rng, [3, 1, 0, 20], [30, 1, 0, 21], heads, kv, hd, hd, spare=60)
        caches = [Cache(lib, np.random.default_rng(2), pn.BF16, hd, kv, page, [80] * 4) for _ in range(2)]
        outs = [r.outs(pn.F32)[0] for _ in range(2)]

        def call(i):
            lib.g4_kv_page_append(*caches[i].args(), *r.kv_in(), *r.q_in(), outs[i].ptr, heads * hd + 16, pn.F32, *r.turn(),
                                  *r.seqs())

        lib.g4_graph_begin()
        call(0)
        g = C.c_void_p()
        lib.g4_graph_end(C.byref(g))
        for n, lens in (([3, 1, 0, 20], [30, 1, 0, 21]), ([1, 1, 1, 1], [31, 2, 1, 22]), ([0, 7, 10, 5], [31, 9, 11, 27])):
            x = rows(rng, r.m, 1, r.x[0].shape[1])
            r.d[0].write(x)
            r.d[6].write(pn.starts(n))
            r.d[7].write(np.asarray(lens, np.int32))
            lib.g4_graph_launch(g.value)
            call(1)
            lib.g4_sync()
            for a, b in ((outs[0], outs[1]), (caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
                assert same_bits(a.to_array(np.uint8), b.to_array(np.uint8))
        lib.g4_graph_destroy(g.value)
