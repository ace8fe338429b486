"""GPU parity of the paged KV cache (stored, read back), of the attention of one
new token of every sequence over it, and of the attention of packed prompts,
against plain forms in 64 bits (tests/paged_np.py holds them and derives the
bounds).

The cache append is main.c:1901-1904 and the attention block main.c:1909-1950
of the reference, which runs one sequence.
"""
import ctypes as C

import numpy as np
import pytest

import paged_np as pn

pytestmark = pytest.mark.gpu

F = C.c_float
NAN = np.float32(np.nan)


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


def dbuf(lib, a):
    from g4 import DBuf
    return DBuf.from_array(lib, np.ascontiguousarray(a))


def filled(lib, nbytes, byte=0xFF):
    """device bytes all set: NaN in every type, codes -1"""
    from g4 import DBuf
    b = DBuf(lib, nbytes)
    lib.g4_memset(b.ptr, byte, nbytes)
    return b


class Cache:
    """two pools and the pages of a batch of sequences"""

    def __init__(self, lib, rng, kind, hd, n_kv, page, lens, table=None, pages=None, extra=2):
        """extra: table entries past the longest sequence's; many of them and the work is split whatever the lengths"""
        self.lib, self.kind, self.hd, self.n_kv, self.page = lib, kind, hd, n_kv, page
        if table is None:
            table, pages = pn.page_table(rng, lens, page, extra=extra)
        self.table, self.pages = np.ascontiguousarray(table, np.int32), pages
        size = lib.L.g4_kv_pool_bytes(kind, pages, page, n_kv, hd)
        self.k, self.v = filled(lib, size), filled(lib, size)
        self.dtable = dbuf(lib, self.table)

    def args(self):
        return (self.k.ptr, self.v.ptr, self.kind, self.pages, self.page, self.n_kv, self.hd, self.dtable.ptr,
                self.table.shape[1])

    def store(self, k, v, n, lens, m=None, stride=None):
        """rows k, v [m, stride floats] of n[s] rows a sequence"""
        dk, dv, cu, dl = (dbuf(self.lib, a) for a in (k, v, pn.starts(n), np.asarray(lens, np.int32)))
        self.lib.g4_kv_page_store(*self.args(), dk.ptr, dv.ptr, stride or k.shape[1], cu.ptr, dl.ptr, len(n),
                                  m or k.shape[0])
        self.lib.g4_sync()

    def load(self, n, lens, pad=0, stride=None):
        w = stride or self.n_kv * self.hd
        rows = sum(n) + pad
        dk, dv = filled(self.lib, rows * w * 4, 0x3F), filled(self.lib, rows * w * 4, 0x3F)
        cu, dl = dbuf(self.lib, pn.starts(n)), dbuf(self.lib, np.asarray(lens, np.int32))
        self.lib.g4_kv_page_load(*self.args(), dk.ptr, dv.ptr, w, cu.ptr, dl.ptr, len(n), rows)
        return tuple(d.to_array(np.float32).reshape(rows, w) for d in (dk, dv))


def rows(rng, m, heads, hd):
    return rng.standard_normal((m, heads * hd)).astype(np.float32)


def same(a, b):
    """equal values (signed zeros alike), NaN where NaN"""
    return np.array_equal(a, b, equal_nan=True)


def within(err, bound, at):
    worst = float(np.max(err / bound))
    assert worst <= 1.0, (at, worst)


UNTOUCHED = np.full(1, 0x3F3F3F3F, np.uint32).view(np.float32)[0]


@pytest.mark.parametrize("kind", pn.TYPES)
@pytest.mark.parametrize("hd,n_kv,page", [(64, 3, 16), (128, 1, 32), (256, 2, 64), (512, 2, 16), (256, 1, 4096)])
def test_store_load(lib, kind, hd, n_kv, page):
    """Ragged turns appended one after the other, read back whole: lengths of 0
    and 1, pages and blocks that end inside a turn, rows past the last sequence
    and strides wider than the rows."""
    rng = np.random.default_rng(hd + page)
    turns = [[5, 0, 1, 33, 16, 64, 2], [1, 1, 1, 1, 1, 1, 1], [0, 40, 15, 0, 31, 17, 14]]
    total = np.sum(turns, 0)
    c = Cache(lib, rng, kind, hd, n_kv, page, total)
    had = np.zeros(7, int)
    w = n_kv * hd
    all_k, all_v = [[[] for _ in range(7)] for _ in range(2)]
    for n in turns:
        m, stride = sum(n) + 3, w + 8
        k, v = rows(rng, m, 1, stride), rows(rng, m, 1, stride)
        k[-3:] = v[-3:] = NAN
        had = had + n
        c.store(k, v, n, had, m=m)
        at = 0
        for s, t in enumerate(n):
            all_k[s].append(k[at:at + t, :w])
            all_v[s].append(v[at:at + t, :w])
            at += t
    wk, wv = (np.concatenate([r for s in a for r in s]) for a in (all_k, all_v))
    for pad, stride in ((0, None), (4, w + 12)):
        gk, gv = c.load(list(total), total, pad=pad, stride=stride)
        n = sum(total)
        for got, want in ((gk, wk), (gv, wv)):
            assert same(got[:n, :w], pn.held(want, kind, hd))
            assert (got[n:] == UNTOUCHED).all() and (got[:, w:] == UNTOUCHED).all()
    # the last rows of each sequence only
    last = [min(int(t), 9) for t in total]
    gk, gv = c.load(last, total)
    pick = np.concatenate([np.arange(e - t, e) for t, e in zip(last, np.cumsum(total))])
    assert same(gk, pn.held(wk[pick], kind, hd)) and same(gv, pn.held(wv[pick], kind, hd))


@pytest.mark.parametrize("kind", pn.TYPES)
def test_store_leaves_others(lib, kind):
    """A store changes the new positions only: every byte of the pools that
    belongs to another position stays."""
    rng = np.random.default_rng(3)
    hd, n_kv, page = 128, 2, 32
    lens = [70, 41]
    c = Cache(lib, rng, kind, hd, n_kv, page, [96, 96])
    full = rows(rng, 192, n_kv, hd)
    c.store(full, full[::-1].copy(), [96, 96], [96, 96])
    before = [np.split(a, 2) for a in c.load([96, 96], [96, 96])]
    new = rows(rng, 12, n_kv, hd)
    c.store(new, -new, [7, 5], lens)
    after = [np.split(a, 2) for a in c.load([96, 96], [96, 96])]
    for i, sign in ((0, 1), (1, -1)):
        for s, n in ((0, 7), (1, 5)):
            rows_new = new[:7] if s == 0 else new[7:]
            want = before[i][s].copy()
            want[lens[s] - n:lens[s]] = pn.held(sign * rows_new, kind, hd)
            assert same(after[i][s], want)


def test_q8_rows(lib):
    """Quantisation's edges: zero rows, subnormal and huge rows, ties, one large
    element, an infinity or NaN (the whole head reads NaN, its neighbours not)."""
    rng = np.random.default_rng(4)
    hd, n_kv = 256, 2
    x = rows(rng, 16, n_kv, hd)
    x[0] = 0
    x[1] *= np.float32(1e-44)
    x[2] *= np.float32(7e37)
    x[3, :hd] = np.float32(0.5) * (np.arange(hd) % 255 - 127)     # d = 0.5: codes exact
    x[4, :hd] = np.arange(hd) - 127.5                                # nothing exact
    x[5, 7] = 1e6
    x[6, 3] = np.inf
    x[7, hd + 4] = -np.inf
    x[8, hd - 1] = np.nan
    x[9] = -0.0
    x[10, :hd] = np.where(np.arange(hd) == 0, 127, 0.5 + np.arange(hd) % 100)   # d = 1: ties
    c = Cache(lib, rng, pn.Q8, hd, n_kv, 16, [16])
    c.store(x, x[::-1].copy(), [16], [16])
    gk, gv = c.load([16], [16])
    assert same(gk, pn.held(x, pn.Q8, hd)) and same(gv, pn.held(x[::-1], pn.Q8, hd))
    assert np.isnan(gk[6, :hd]).all() and np.isfinite(gk[6, hd:]).all()


def test_half_rows(lib):
    """16-bit caches keep infinities and NaN, round to even and, fp16, overflow to infinity"""
    rng = np.random.default_rng(5)
    x = rows(rng, 16, 1, 64)
    x[0, :6] = [np.inf, -np.inf, np.nan, 65519.9, 65520.0, 1e-8]
    x[1, :4] = [1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8]
    for kind in (pn.F16, pn.BF16, pn.F32):
        c = Cache(lib, rng, kind, 64, 1, 16, [16])
        c.store(x, -x, [16], [16])
        gk, gv = c.load([16], [16])
        assert same(gk, pn.held(x, kind, 64)) and same(gv, pn.held(-x, kind, 64))


def test_rows_that_do_not_fit(lib):
    """Sequences whose lengths do not fit and pages outside the pool: skipped,
    dropped, read as NaN; their neighbours are not touched."""
    rng = np.random.default_rng(6)
    hd, n_kv, page = 64, 1, 16
    table = np.array([[0, 1], [2, 99], [3, 4], [-7, 5], [6, 7]], np.int32)
    c = Cache(lib, rng, pn.F32, hd, n_kv, page, None, table=table, pages=8)
    n = [20, 32, 33, 32, 10]
    lens = np.array([20, 32, 33, 32, 9], np.int32)      # 2: past the table; 4: fewer than its rows
    x = rows(rng, sum(n), n_kv, hd)
    c.store(x, x, n, lens)
    gk, _ = c.load(n, lens)
    at = pn.starts(n)
    part = [gk[at[s]:at[s + 1]] for s in range(5)]
    want = [x[at[s]:at[s + 1]] for s in range(5)]
    assert same(part[0], want[0])
    assert same(part[1][:16], want[1][:16]) and np.isnan(part[1][16:]).all()
    assert (part[2] == UNTOUCHED).all() and (part[4] == UNTOUCHED).all()
    assert np.isnan(part[3][:16]).all() and same(part[3][16:], want[3][16:])
    # row starts that are not ascending or run past m: those sequences are skipped
    good = rows(rng, 8, n_kv, hd)
    c2 = Cache(lib, rng, pn.F32, hd, n_kv, page, [16] * 4)
    dk, dl = dbuf(lib, good), dbuf(lib, np.array([16, 16, 16, 16], np.int32))
    old = rows(rng, 64, n_kv, hd)
    c2.store(old, old, [16] * 4, [16] * 4)
    before, _ = c2.load([16] * 4, [16] * 4)
    cu = dbuf(lib, np.array([0, 4, 3, -2, 200], np.int32))
    lib.g4_kv_page_store(*c2.args(), dk.ptr, dk.ptr, hd, cu.ptr, dl.ptr, 4, 8)
    after, _ = c2.load([16] * 4, [16] * 4)
    assert same(after[16:], before[16:])


def run_decode(lib, c, q, lens, n_heads, window, scale, q_stride=None, out_stride=None):
    n, hd = len(lens), c.hd
    dq, dl = dbuf(lib, q), dbuf(lib, np.asarray(lens, np.int32))
    os = out_stride or n_heads * hd
    out = filled(lib, n * os * 4, 0x3F)
    part = filled(lib, lib.L.g4_attn_decode_paged_part_bytes(n_heads, c.n_kv, hd))
    lib.g4_attn_decode_paged(dq.ptr, q.shape[1], *c.args(), dl.ptr, n, window, n_heads, F(scale), part.ptr, out.ptr, os)
    return out.to_array(np.float32).reshape(n, os)


def check_decode(lib, seed, kind, hd, n_heads, n_kv, page, lens, window=0, scale=None, gain=3.0, extra=0):
    rng = np.random.default_rng(seed)
    scale = hd ** -0.5 if scale is None else scale
    c = Cache(lib, rng, kind, hd, n_kv, page, lens)
    k, v = rows(rng, sum(lens), n_kv, hd), rows(rng, sum(lens), n_kv, hd)
    if sum(lens):
        c.store(k, v, list(lens), lens)
    q = rows(rng, len(lens), 1, n_heads * hd + extra) * np.float32(gain)
    got = run_decode(lib, c, q, lens, n_heads, window, scale, out_stride=n_heads * hd + extra)
    at = pn.starts(lens)
    hk, hv = pn.held(k, kind, hd), pn.held(v, kind, hd)
    for s, t in enumerate(lens):
        o = got[s, :n_heads * hd].reshape(n_heads, hd)
        if t == 0:
            assert (o == 0).all(), s
            continue
        first = max(0, t - window) if window else 0
        want, bound = pn.attention(q[s:s + 1, :n_heads * hd].reshape(1, n_heads, hd),
                                   hk[at[s]:at[s + 1]].reshape(t, n_kv, hd), hv[at[s]:at[s + 1]].reshape(t, n_kv, hd),
                                   [first], scale)
        err = np.abs(o - want[0])
        within(err, bound[0], (s, t))
    if extra:
        assert (got[:, n_heads * hd:] == UNTOUCHED).all()


@pytest.mark.parametrize("kind", pn.TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_decode_types(lib, kind, hd):
    """every cache type and head_dim, ragged lengths with 0 and 1 among them"""
    check_decode(lib, 10 + hd, kind, hd, 8, 2, 16, [1, 0, 15, 16, 17, 31, 33, 64, 65, 100, 257, 0, 700])


@pytest.mark.parametrize("n_heads,n_kv", [(1, 1), (3, 3), (8, 1), (10, 2), (12, 1), (16, 1), (24, 8), (17, 1), (40, 2)])
def test_decode_heads(lib, n_heads, n_kv):
    """one head to twenty heads on a kv head"""
    for kind, hd in ((pn.BF16, 128), (pn.Q8, 256)):
        check_decode(lib, 30 + n_heads, kind, hd, n_heads, n_kv, 32, [5, 130, 64, 1])


@pytest.mark.parametrize("window", [1, 7, 64, 100, 512, 5000])
def test_decode_window(lib, window):
    """windows that end inside a block, at one and past the length; pages before the window have been given away"""
    lens = [1, 6, 63, 64, 65, 400, 1025]
    for kind, hd, page in ((pn.F32, 256, 16), (pn.Q8, 64, 64)):
        check_decode(lib, 50 + window, kind, hd, 4, 2, page, lens, window=window)


def test_decode_window_pages_gone(lib):
    """entries of pages that lie wholly before the window are never read"""
    rng = np.random.default_rng(60)
    hd, n_kv, page, t, w = 128, 1, 16, 200, 50
    c = Cache(lib, rng, pn.BF16, hd, n_kv, page, [t])
    k, v = rows(rng, t, n_kv, hd), rows(rng, t, n_kv, hd)
    c.store(k, v, [t], [t])
    q = rows(rng, 1, 2, hd)
    a = run_decode(lib, c, q, [t], 2, w, 0.1)
    c.table[0, :(t - w) // page] = -1
    c.dtable = dbuf(lib, c.table)
    b = run_decode(lib, c, q, [t], 2, w, 0.1)
    assert np.isfinite(a).all() and same(a, b)


@pytest.mark.parametrize("kind,hd", [(pn.BF16, 256), (pn.Q8, 512), (pn.F32, 64)])
def test_decode_long(lib, kind, hd):
    """one long sequence, split over many workgroups, beside short ones"""
    check_decode(lib, 70, kind, hd, 4, 1, 64, [3, 20011, 0, 129])


def test_decode_many(lib):
    """more sequences than workgroups, short throughout and with some long ones; the most there may be"""
    rng = np.random.default_rng(71)
    check_decode(lib, 71, pn.BF16, 64, 2, 2, 16, [int(x) for x in rng.integers(0, 40, 700)])
    check_decode(lib, 71, pn.BF16, 64, 2, 2, 16, [int(x) for x in rng.integers(0, 40, 300)] + [900, 0, 1300])
    check_decode(lib, 71, pn.Q8, 64, 1, 1, 16, [int(x) for x in rng.integers(0, 6, 4095)] + [700])


def test_decode_splits(lib):
    """numbers of tiles on either side of what one workgroup, all of them and one round take"""
    for lens in ([32 * 511], [32 * 512 + 1], [32 * 513], [32 * 2048 - 31], [33] * 64, [65] * 65, [300] * 33, [1] * 63 + [5000]):
        check_decode(lib, 79, pn.BF16, 64, 1, 1, 64, lens, window=0, gain=1.0)


@pytest.mark.parametrize("kind,hd", [(pn.F32, 64), (pn.F32, 512), (pn.BF16, 256), (pn.BF16, 512), (pn.Q8, 128), (pn.Q8, 512)])
def test_decode_whole_or_split(lib, kind, hd):
    """tables and windows on either side of the keys up to which a workgroup takes a sequence whole"""
    for most in (128, 256, 512):
        check_decode(lib, 80, kind, hd, 8, 2, 16, [most - 33, most - 1, 1, 90])              # 16 or 32 entries past it
        check_decode(lib, 81, kind, hd, 8, 2, 16, [most - 32, 0, 17], window=0)
        for w in (most, most + 1):
            check_decode(lib, 82, kind, hd, 8, 2, 32, [700, most, most + 1, 5], window=w)


def test_decode_split_extremes(lib):
    """what the tests of heads and of extremes see, beside a sequence too long to be taken whole"""
    for kind in (pn.F32, pn.BF16, pn.Q8):
        check_decode(lib, 83, kind, 128, 4, 2, 16, [50, 300, 900], gain=60.0, scale=1.0)
        check_decode(lib, 84, kind, 128, 4, 2, 16, [50, 300, 900], gain=0.0, scale=1.0)
        check_decode(lib, 85, kind, 128, 4, 2, 16, [50, 300, 900], scale=-0.09)
    for n_heads, n_kv in ((1, 1), (12, 1), (17, 1), (40, 2)):
        for kind, hd in ((pn.BF16, 128), (pn.Q8, 256)):
            check_decode(lib, 86 + n_heads, kind, hd, n_heads, n_kv, 32, [5, 130, 900, 64, 1])
            check_decode(lib, 87 + n_heads, kind, hd, n_heads, n_kv, 32, [5, 130, 900, 64, 1], window=600)


def test_decode_strides(lib):
    """q and out rows wider than their heads"""
    check_decode(lib, 72, pn.F16, 256, 8, 2, 32, [40, 3, 77], extra=12)


@pytest.mark.parametrize("extra", [2, 40])
def test_decode_pages_outside(lib, extra):
    """a page outside the pool or a length past the table: NaN in that sequence's row and nowhere else"""
    rng = np.random.default_rng(73)
    hd, page = 64, 16
    for kind in pn.TYPES:
        c = Cache(lib, rng, kind, hd, 1, page, [40, 40, 40, 40], extra=extra)
        x = rows(rng, 160, 1, hd)
        c.store(x, x, [40] * 4, [40] * 4)
        q = rows(rng, 4, 2, hd)
        a = run_decode(lib, c, q, [40, 40, 40, 40], 2, 0, 0.2)
        c.table[1, 1] = c.pages
        c.table[2, 2] = -1
        c.dtable = dbuf(lib, c.table)
        b = run_decode(lib, c, q, [40, 40, 40, c.table.shape[1] * page + 1], 2, 0, 0.2)
        assert same(a[0], b[0]) and np.isnan(b[1:]).all()
        d = run_decode(lib, c, q, [40, 16, -3, 40], 2, 0, 0.2)
        assert same(d[0], a[0]) and np.isfinite(d[1]).all() and np.isnan(d[2]).all() and same(d[3], a[3])


@pytest.mark.parametrize("extra", [2, 40])
@pytest.mark.parametrize("kind", [pn.F32, pn.F16, pn.BF16])
def test_decode_not_finite(lib, kind, extra):
    """infinities and NaN at positions that are not seen change nothing; seen, they make their heads NaN or
    infinite and no others"""
    rng = np.random.default_rng(74)
    hd, n_kv, page, t = 128, 2, 32, 90
    c = Cache(lib, rng, kind, hd, n_kv, page, [128, 128], extra=extra)
    k, v = rows(rng, 256, n_kv, hd), rows(rng, 256, n_kv, hd)
    k2, v2 = k.copy(), v.copy()
    for a in (k2, v2):      # past the length, before the window
        a[t:128] = NAN
        a[t + 1] = np.inf
        a[:10] = -np.inf
    q = rows(rng, 2, 4, hd)
    c.store(k, v, [128, 128], [128, 128])
    want = run_decode(lib, c, q, [t, 128], 4, 80, 0.1)
    c.store(k2, v2, [128, 128], [128, 128])
    assert same(run_decode(lib, c, q, [t, 128], 4, 80, 0.1), want)
    k2[50, :5] = NAN        # seen by the heads of kv head 0 in sequence 0
    c.store(k2, v2, [128, 128], [128, 128])
    got = run_decode(lib, c, q, [t, 128], 4, 80, 0.1).reshape(2, 4, hd)
    want = want.reshape(2, 4, hd)
    assert np.isnan(got[0, :2]).all() and same(got[0, 2:], want[0, 2:]) and same(got[1], want[1])


def test_decode_extremes(lib):
    """scores far apart (one key takes all), all equal, large magnitudes of K and V, a negative scale"""
    for kind in (pn.F32, pn.BF16, pn.Q8):
        check_decode(lib, 75, kind, 128, 4, 2, 16, [50, 300], gain=60.0, scale=1.0)
        check_decode(lib, 76, kind, 128, 4, 2, 16, [50, 300], gain=0.0, scale=1.0)
        check_decode(lib, 77, kind, 128, 4, 2, 16, [50, 300], scale=-0.09)
    check_decode(lib, 78, pn.BF16, 256, 4, 2, 16, [50, 300], gain=1e-18, scale=1e17)


NPT = {pn.F32: np.float32, pn.F16: np.float16, pn.BF16: np.uint16}


def cast(x, kind):
    """(array of the type's bits, its values in float32)"""
    if kind == pn.BF16:
        b = pn.bf16_bits(x)
        return b, pn.bf16_back(b)
    y = x.astype(NPT[kind])
    return y, y.astype(np.float32)


def run_prompt(lib, q, k, v, kind, cu, m, window, n_heads, n_kv, hd, scale, out_stride=None):
    """rows of the type's bits -> (out bits, out as float32); out starts as 0x3F3F..."""
    es = q.dtype.itemsize
    os = out_stride or n_heads * hd
    out = filled(lib, m * os * es, 0x3F)
    dq, dk, dv, dcu = (dbuf(lib, a) for a in (q, k, v, np.asarray(cu, np.int32)))
    n = len(cu) - 1
    work = filled(lib, lib.L.g4_attn_prompt_packed_work_bytes(kind, n, m, n_kv, hd))
    lib.g4_attn_prompt_packed(dq.ptr, q.shape[1], dk.ptr, dv.ptr, k.shape[1], out.ptr, os, kind, dcu.ptr, n, m, window,
                              n_heads, n_kv, hd, F(scale), work.ptr)
    bits = out.to_array(NPT[kind]).reshape(m, os)
    return bits, (pn.bf16_back(bits) if kind == pn.BF16 else bits.astype(np.float32))


def check_prompt(lib, seed, kind, hd, n_heads, n_kv, n, window=0, scale=None, gain=2.0, pad=0, extra=0, some=None):
    rng = np.random.default_rng(seed)
    scale = hd ** -0.5 if scale is None else scale
    m, cu = sum(n) + pad, pn.starts(n)
    q, qf = cast(rows(rng, m, 1, n_heads * hd + extra) * np.float32(gain), kind)
    k, kf = cast(rows(rng, m, 1, n_kv * hd + extra), kind)
    v, vf = cast(rows(rng, m, 1, n_kv * hd + extra), kind)
    bits, got = run_prompt(lib, q, k, v, kind, cu, m, window, n_heads, n_kv, hd, scale, out_stride=n_heads * hd + extra)
    for s, t in enumerate(n):
        for lo in range(0, t, 128):
            hi = min(t, lo + 128)
            if some is not None and lo and hi < t and lo // 128 % some:
                continue
            first = [max(0, i + 1 - window) if window else 0 for i in range(lo, hi)]
            r = slice(cu[s] + lo, cu[s] + hi)
            kk = slice(cu[s], cu[s] + hi)
            want, bound = pn.attention(qf[r, :n_heads * hd].reshape(hi - lo, n_heads, hd),
                                       kf[kk, :n_kv * hd].reshape(hi, n_kv, hd), vf[kk, :n_kv * hd].reshape(hi, n_kv, hd),
                                       first, scale)
            if kind != pn.F32:
                # weights rounded to the type once (each off by HALF of itself: of sum p |v|, which is at most
                # max |v|, and by the smallest subnormal's half at a maximum of 1) and the result rounded to it
                big = np.abs(vf[kk, :n_kv * hd]).max()
                bound = bound + pn.HALF[kind] * (np.abs(want) + 1.01 * big) + 2.0 ** -25 * hi * big
            err = np.abs(got[r, :n_heads * hd].reshape(hi - lo, n_heads, hd) - want)
            within(err, bound, (s, lo))
    untouched = np.full(1, 0x3F3F3F3F, np.uint32).view(bits.dtype)[0]
    assert (bits[sum(n):] == untouched).all() and (bits[:, n_heads * hd:] == untouched).all()


@pytest.mark.parametrize("kind", [pn.F32, pn.F16, pn.BF16])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_prompt_types(lib, kind, hd):
    """every type and head_dim; sequences of 0, 1 and odd lengths, rows past the last one"""
    check_prompt(lib, 100 + hd, kind, hd, 8, 2, [1, 0, 31, 32, 33, 0, 70, 129, 2], pad=5)


@pytest.mark.parametrize("n_heads,n_kv", [(1, 1), (3, 3), (5, 1), (8, 1), (10, 2), (12, 1), (24, 8), (20, 1)])
def test_prompt_heads(lib, n_heads, n_kv):
    for kind, hd in ((pn.F32, 128), (pn.BF16, 64)):
        check_prompt(lib, 120 + n_heads, kind, hd, n_heads, n_kv, [40, 1, 65, 100])


@pytest.mark.parametrize("window", [1, 5, 32, 64, 100, 512])
def test_prompt_window(lib, window):
    for kind, hd in ((pn.F32, 256), (pn.F16, 128), (pn.BF16, 512)):
        check_prompt(lib, 140 + window, kind, hd, 4, 2, [3, 96, 150, 33], window=window)


@pytest.mark.parametrize("kind,hd,window", [(pn.F32, 256, 512), (pn.F32, 512, 0), (pn.BF16, 256, 0), (pn.F16, 128, 300)])
def test_prompt_long(lib, kind, hd, window):
    """thousands of rows, the first, the last and some between them checked"""
    check_prompt(lib, 150, kind, hd, 2, 1, [1500, 2777], window=window, some=8)


def test_prompt_strides(lib):
    for kind in (pn.F32, pn.F16, pn.BF16):
        check_prompt(lib, 160, kind, 128, 4, 2, [50, 7], extra=8, pad=2)


def test_prompt_many(lib):
    """hundreds of short sequences"""
    rng = np.random.default_rng(161)
    check_prompt(lib, 161, pn.BF16, 64, 2, 1, [int(x) for x in rng.integers(0, 9, 600)])


def test_prompt_extremes(lib):
    """weights on one key, equal weights, a negative scale, magnitudes far from 1"""
    for kind in (pn.F32, pn.BF16):
        check_prompt(lib, 162, kind, 128, 4, 2, [150], gain=60.0, scale=1.0)
        check_prompt(lib, 163, kind, 128, 4, 2, [150], gain=0.0, scale=1.0)
        check_prompt(lib, 164, kind, 128, 4, 2, [150], scale=-0.09)
        check_prompt(lib, 165, kind, 128, 4, 2, [150], gain=1e-18, scale=1e17)


@pytest.mark.parametrize("kind", [pn.F32, pn.F16, pn.BF16])
def test_prompt_not_finite(lib, kind):
    """infinities and NaN in rows of other sequences, in rows past the last sequence and in later rows of the same
    sequence change no row that does not see them; a row that sees them has NaN in the heads that do"""
    rng = np.random.default_rng(166)
    hd, n_heads, n_kv, n = 128, 4, 2, [50, 45, 20]
    m, cu = sum(n) + 6, pn.starts(n)
    q, k, v = (rows(rng, m, h, hd) for h in (n_heads, n_kv, n_kv))
    a = run_prompt(lib, *(cast(x, kind)[0] for x in (q, k, v)), kind, cu, m, 0, n_heads, n_kv, hd, 0.1)[1]
    k[cu[3]:] = v[cu[3]:] = q[cu[3]:] = NAN
    v[50 + 37, hd + 3] = np.inf         # row 37 of sequence 1, kv head 1
    k[50 + 40, 5] = NAN                 # row 40, kv head 0
    b = run_prompt(lib, *(cast(x, kind)[0] for x in (q, k, v)), kind, cu, m, 0, n_heads, n_kv, hd, 0.1)[1]
    a, b = (x.reshape(m, n_heads, hd) for x in (a, b))
    assert same(a[:87, 2:], b[:87, 2:]) and same(a[:90, :2], b[:90, :2])
    assert same(a[95:115], b[95:115])
    assert not np.isfinite(b[87:95, 2:, 3]).any() and np.isnan(b[90:95, :2]).all()


def test_prompt_starts_that_do_not_fit(lib):
    """row starts that are not ascending or run past m: those sequences' rows are left as they are"""
    rng = np.random.default_rng(167)
    hd, m = 64, 40
    q, k, v = (rows(rng, m, 2, hd) for _ in range(3))
    bits, got = run_prompt(lib, q, k, v, pn.F32, [0, 10, 300, 290, -5], m, 0, 2, 2, hd, 0.1)
    assert (got[10:] == UNTOUCHED).all()
    want, bound = pn.attention(q[:10].reshape(10, 2, hd), k[:10].reshape(10, 2, hd), v[:10].reshape(10, 2, hd), [0] * 10, 0.1)
    assert (np.abs(got[:10].reshape(10, 2, hd) - want) <= bound).all() or (got[:10] == UNTOUCHED).all()


def test_serving(lib):
    """The operators as a server uses them: prompts of a ragged batch (attention, cache written), then steps of
    one token each; every output equals a plain forward over the whole sequences."""
    rng = np.random.default_rng(200)
    hd, n_heads, n_kv, page, window, scale = 256, 8, 2, 16, 100, 1 / 16
    n, steps = [37, 1, 130, 64], 20
    lens = np.array(n)
    total = [t + steps for t in n]
    seqs = [tuple(rows(rng, t, h, hd) for h in (n_heads, n_kv, n_kv)) for t in total]
    for kind in pn.TYPES:
        c = Cache(lib, rng, kind, hd, n_kv, page, total)
        q, k, v = (np.concatenate([s[i][:t] for s, t in zip(seqs, n)]) for i in range(3))
        got = [[x] for x in np.split(run_prompt(lib, q, k, v, pn.F32, pn.starts(n), len(q), window, n_heads, n_kv, hd,
                                                scale)[1], pn.starts(n)[1:-1])]
        c.store(k, v, n, n)
        for i in range(steps):
            q, k, v = (np.stack([s[j][t + i] for s, t in zip(seqs, n)]) for j in range(3))
            c.store(k, v, [1] * 4, lens + i + 1)
            o = run_decode(lib, c, q, lens + i + 1, n_heads, window, scale)
            for s in range(4):
                got[s].append(o[s:s + 1])
        gk, _ = c.load(total, total)
        assert same(gk, pn.held(np.concatenate([s[1] for s in seqs]), kind, hd))
        for s, t in enumerate(n):
            qs, ks, vs = seqs[s]
            o = np.concatenate(got[s]).reshape(total[s], n_heads, hd)
            hk, hv = pn.held(ks, kind, hd), pn.held(vs, kind, hd)
            first = [max(0, i + 1 - window) for i in range(total[s])]
            want, bound = pn.attention(qs[:t].reshape(t, n_heads, hd), ks[:t].reshape(t, n_kv, hd),
                                       vs[:t].reshape(t, n_kv, hd), first[:t], scale)
            assert (np.abs(o[:t] - want) <= bound).all()
            want, bound = pn.attention(qs[t:].reshape(steps, n_heads, hd), hk.reshape(-1, n_kv, hd),
                                       hv.reshape(-1, n_kv, hd), first[t:], scale)
            assert (np.abs(o[t:] - want) <= bound).all()


def same_bits(a, b):
    return np.array_equal(a.view(np.uint8), b.view(np.uint8))


class Stream:
    """work on a created library stream"""

    def __init__(self, lib):
        self.lib = lib

    def __enter__(self):
        p = C.c_void_p()
        self.lib.g4_stream_create(C.byref(p))
        self.p = p.value
        self.lib.g4_set_stream(self.p)
        return self

    def __exit__(self, *exc):
        self.lib.g4_sync()
        self.lib.g4_set_stream(None)
        self.lib.g4_stream_destroy(self.p)


@pytest.mark.parametrize("kind", [pn.BF16, pn.Q8])
def test_graph_of_steps(lib, kind):
    """A step (store, decode attention) captured once and replayed while the lengths grow: every replay equals the
    eager calls bit for bit, the program's own work running in between."""
    rng = np.random.default_rng(300)
    hd, n_heads, n_kv, page, steps = 128, 8, 2, 16, 6
    n = [0, 33, 500, 14]
    total = [t + steps for t in n]
    table, pages = pn.page_table(rng, total, page)
    hist = rows(rng, sum(n), n_kv, hd)
    step = [(rows(rng, 4, n_heads, hd), rows(rng, 4, n_kv, hd), rows(rng, 4, n_kv, hd)) for _ in range(steps)]
    results = []
    for captured in (False, True):
        with Stream(lib):
            c = Cache(lib, rng, kind, hd, n_kv, page, None, table=table, pages=pages)
            c.store(hist, hist[::-1].copy(), n, n)
            dq, dk, dv = (filled(lib, a.nbytes) for a in step[0])
            lens, cu = filled(lib, 16), dbuf(lib, pn.starts([1] * 4))
            out = filled(lib, 4 * n_heads * hd * 4)
            part = filled(lib, lib.L.g4_attn_decode_paged_part_bytes(n_heads, n_kv, hd))

            def run():
                lib.g4_kv_page_store(*c.args(), dk.ptr, dv.ptr, n_kv * hd, cu.ptr, lens.ptr, 4, 4)
                lib.g4_attn_decode_paged(dq.ptr, n_heads * hd, *c.args(), lens.ptr, 4, 200, n_heads, F(0.1), part.ptr,
                                         out.ptr, n_heads * hd)

            graph = None
            if captured:
                lens.write(np.array(total, np.int32))
                lib.g4_graph_begin()
                run()
                g = C.c_void_p()
                lib.g4_graph_end(C.byref(g))
                graph = g.value
            got = []
            for i, (q, k, v) in enumerate(step):
                dq.write(q)
                dk.write(k)
                dv.write(v)
                lens.write(np.array([t + i + 1 for t in n], np.int32))
                if graph:
                    lib.g4_graph_launch(graph)
                else:
                    run()
                lib.g4_sync()
                got.append(out.to_array(np.float32))
                c.load([t + i + 1 for t in n], [t + i + 1 for t in n])
            results.append(np.stack(got))
            if graph:
                lib.g4_graph_destroy(graph)
    assert np.isfinite(results[0]).all() and same_bits(*results)


@pytest.mark.parametrize("kind,hd", [(pn.F32, 256), (pn.BF16, 256), (pn.F32, 512), (pn.F16, 512), (pn.BF16, 64)])
def test_graph_of_prompts(lib, kind, hd):
    """A prompt batch captured once and replayed with other prompts and other lengths: each replay equals the eager call"""
    rng = np.random.default_rng(301)
    n_heads, n_kv, m, scale = 8, 2, 420, 0.07
    es = 4 if kind == pn.F32 else 2
    batches = [[200, 219, 1], [420, 0, 0], [33, 300, 60], [0, 5, 0]]
    data = [tuple(cast(rows(rng, m, h, hd), kind)[0] for h in (n_heads, n_kv, n_kv)) for _ in batches]
    with Stream(lib):
        dq, dk, dv = (filled(lib, a.nbytes) for a in data[0])
        cu, out = filled(lib, 16), filled(lib, m * n_heads * hd * es)
        work = filled(lib, lib.L.g4_attn_prompt_packed_work_bytes(kind, 3, m, n_kv, hd))

        def run():
            lib.g4_attn_prompt_packed(dq.ptr, n_heads * hd, dk.ptr, dv.ptr, n_kv * hd, out.ptr, n_heads * hd, kind, cu.ptr, 3,
                                      m, 100, n_heads, n_kv, hd, F(scale), work.ptr)

        def batch(i, call):
            for d, a in zip((dq, dk, dv), data[i]):
                d.write(a)
            cu.write(pn.starts(batches[i]))
            lib.g4_memset(out.ptr, 0x3F, out.nbytes)
            call()
            lib.g4_sync()
            return out.to_array(np.uint8)

        want = [batch(i, run) for i in range(len(batches))]
        cu.write(pn.starts(batches[0]))
        lib.g4_graph_begin()
        run()
        g = C.c_void_p()
        lib.g4_graph_end(C.byref(g))
        for i in (2, 0, 1, 3, 2):
            assert same_bits(batch(i, lambda: lib.g4_graph_launch(g.value)), want[i]), i
        lib.g4_graph_destroy(g.value)


def test_calls_one_after_the_other(lib):
    """Calls of other sizes that share part and work, none of which waits: each result is its own"""
    rng = np.random.default_rng(302)
    hd, n_kv, n_heads, page = 128, 2, 8, 32
    part = filled(lib, lib.L.g4_attn_decode_paged_part_bytes(n_heads, n_kv, hd))
    cases = []
    for lens in ([4000, 3], [70], [0, 0, 900], [1]):
        c = Cache(lib, rng, pn.F16, hd, n_kv, page, lens)
        x = rows(rng, sum(lens), n_kv, hd)
        c.store(x, x, lens, lens)
        q = rows(rng, len(lens), n_heads, hd)
        cases.append((c, dbuf(lib, q), dbuf(lib, np.array(lens, np.int32)), filled(lib, q.nbytes),
                      run_decode(lib, c, q, lens, n_heads, 0, 0.1)))
    for _ in range(3):
        for c, dq, dl, out, _want in cases:
            lib.g4_attn_decode_paged(dq.ptr, n_heads * hd, *c.args(), dl.ptr, dl.nbytes // 4, 0, n_heads, F(0.1), part.ptr,
                                     out.ptr, n_heads * hd)
    lib.g4_sync()
    for c, dq, dl, out, want in cases:
        assert same_bits(out.to_array(np.float32).reshape(want.shape), want)


def test_offsets_past_32_bits(lib):
    """pages at the end of pools of 5 GB and more"""
    rng = np.random.default_rng(303)
    for kind, hd, n_kv, page, pages in ((pn.F32, 512, 2, 64, 20000), (pn.Q8, 512, 2, 256, 21000)):
        lens = [150, 61]
        need = [-(-t // page) for t in lens]
        table = np.full((2, max(need)), -1, np.int32)
        at = pages
        for s, c in enumerate(need):
            for i in range(c):
                at -= 1
                table[s, i] = at
        c = Cache(lib, rng, kind, hd, n_kv, page, None, table=table, pages=pages)
        assert c.k.nbytes > 1 << 32
        k, v = rows(rng, sum(lens), n_kv, hd), rows(rng, sum(lens), n_kv, hd)
        c.store(k, v, lens, lens)
        gk, gv = c.load(lens, lens)
        hk, hv = pn.held(k, kind, hd), pn.held(v, kind, hd)
        assert same(gk, hk) and same(gv, hv)
        q = rows(rng, 2, 4, hd)
        got = run_decode(lib, c, q, lens, 4, 0, 0.04).reshape(2, 4, hd)
        cu = pn.starts(lens)
        for s, t in enumerate(lens):
            r = slice(cu[s], cu[s + 1])
            want, bound = pn.attention(q[s].reshape(1, 4, hd), hk[r].reshape(t, n_kv, hd), hv[r].reshape(t, n_kv, hd), [0],
                                       0.04)
            within(np.abs(got[s] - want[0]), bound[0], s)


def test_shared_pages(lib):
    """two sequences with the same first pages (a common prefix) and tails of their own"""
    rng = np.random.default_rng(304)
    hd, n_kv, page = 64, 1, 16
    table = np.array([[0, 1, 2, 3], [0, 1, 4, 5]], np.int32)
    c = Cache(lib, rng, pn.BF16, hd, n_kv, page, None, table=table, pages=6)
    a, b = rows(rng, 50, n_kv, hd), rows(rng, 60, n_kv, hd)
    b[:32] = a[:32]
    c.store(a, a, [50], [50])                       # sequence 0 with the prefix
    second = Cache.__new__(Cache)
    second.__dict__.update(c.__dict__)
    second.table, second.dtable = table[1:], dbuf(lib, table[1:])
    second.store(b[32:], b[32:], [28], [60])        # the other's tail
    gk, gv = c.load([50, 60], [50, 60])
    assert same(gk, pn.held(np.concatenate([a, b]), pn.BF16, hd)) and same(gv, gk)


def test_prompt_lengths(lib):
    """sequences of 1 to 136 rows one after the other, a window that ends inside tiles, three heads on a kv head"""
    for kind in (pn.F32, pn.BF16):
        check_prompt(lib, 305, kind, 64, 6, 2, list(range(1, 141, 9)), window=33)


@pytest.mark.parametrize("hd,window", [(256, 0), (512, 0), (512, 40), (128, 40)])
def test_prompt_magnitudes(lib, hd, window):
    """fp32 rows whose sizes differ by 2^60 from key to key and by 2^20 within a row: what a row does not see, and what
    has next to no weight, costs it no precision, and a key of large scores moves the maximum far at once"""
    rng = np.random.default_rng(400 + hd)
    n_heads, n_kv, n = 4, 2, [300, 130]
    m, cu = sum(n), pn.starts(n)
    q, k, v = (rows(rng, m, h, hd) for h in (n_heads, n_kv, n_kv))
    v *= np.exp2(rng.integers(-30, 31, (m, n_kv * hd // 64))).repeat(64, 1).astype(np.float32)
    v *= np.exp2(rng.integers(-10, 11, v.shape)).astype(np.float32)
    k *= np.exp2(rng.integers(-6, 3, (m, 1))).astype(np.float32)
    k[rng.integers(0, m, 12)] *= np.float32(20)         # scores far from the others', up and down
    v[7] = 0
    v[200] = 0
    k[31] = 0
    scale = hd ** -0.5
    _, got = run_prompt(lib, q, k, v, pn.F32, cu, m, window, n_heads, n_kv, hd, scale)
    for s, t in enumerate(n):
        r = slice(cu[s], cu[s + 1])
        first = [max(0, i + 1 - window) if window else 0 for i in range(t)]
        want, bound = pn.attention(q[r].reshape(t, n_heads, hd), k[r].reshape(t, n_kv, hd), v[r].reshape(t, n_kv, hd), first,
                                   scale)
        # Added for rows this wide: an element of V is met within 2^-39 of its row's largest; and a weight times its V
        # row's power of two is held as two fp16, the largest of them at 2^11 or more (2^15 at most) and each within
        # 2^-25, half of fp16's smallest step: times V's scaled elements, below 2^15, that is 2^-10 a key where the
        # largest key stands for 2^11 * 2^14 at least: 2^-35 of the largest weight * row for each key that is seen.
        big = np.abs(v[r].reshape(t, n_kv, hd)).max(-1).repeat(n_heads // n_kv, 1).astype(np.float64)
        for i in range(t):
            seen = slice(first[i], i + 1)
            for h in range(n_heads):
                sc = scale * (k[r].reshape(t, n_kv, hd)[seen, h // 2].astype(np.float64) @ q[cu[s] + i].reshape(n_heads, hd)[h])
                p = np.exp(sc - sc.max())
                pb = p * big[seen, h]
                bound[i, h] += (2.0 ** -38 * pb.sum() + 2.0 ** -35 * len(p) * pb.max()) / p.sum()
        within(np.abs(got[r].reshape(t, n_heads, hd) - want), bound, s)


@pytest.mark.parametrize("hd", [64, 256])
def test_decode_magnitudes(lib, hd):
    """the same for one token over an fp32 cache, whose products are exact whatever the sizes"""
    rng = np.random.default_rng(410)
    n_heads, n_kv, lens = 4, 2, [300, 1500]
    m = sum(lens)
    k, v = rows(rng, m, n_kv, hd), rows(rng, m, n_kv, hd)
    v *= np.exp2(rng.integers(-30, 31, v.shape)).astype(np.float32)
    k *= np.exp2(rng.integers(-6, 3, (m, 1))).astype(np.float32)
    k[rng.integers(0, m, 12)] *= np.float32(20)
    c = Cache(lib, rng, pn.F32, hd, n_kv, 16, lens)
    c.store(k, v, lens, lens)
    q = rows(rng, 2, n_heads, hd)
    got = run_decode(lib, c, q, lens, n_heads, 0, hd ** -0.5).reshape(2, n_heads, hd)
    cu = pn.starts(lens)
    for s, t in enumerate(lens):
        r = slice(cu[s], cu[s + 1])
        want, bound = pn.attention(q[s].reshape(1, n_heads, hd), k[r].reshape(t, n_kv, hd), v[r].reshape(t, n_kv, hd), [0],
                                   hd ** -0.5)
        within(np.abs(got[s] - want[0]), bound[0], s)
