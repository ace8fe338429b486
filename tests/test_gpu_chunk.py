"""Attention of chunks of new rows over the paged cache (main.c:1909-1950 of the
reference, which has one sequence and one row), against the formula in 64 bits."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import paged_np as pn
from test_gpu_paged import NAN, NPT, Cache, Stream, cast, dbuf, filled, rows, same, same_bits, within

pytestmark = pytest.mark.gpu

F = C.c_float
# types of (rows, cache)
COMBOS = [(pn.F32, pn.F32), (pn.F32, pn.F16), (pn.F32, pn.BF16), (pn.F32, pn.Q8), (pn.F16, pn.F16), (pn.BF16, pn.BF16), (pn.BF16, pn.Q8)]


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


EXTRA = 2


@pytest.fixture(params=[2, 3000], ids=["table", "wide"], autouse=True)
def width(request):
    """entries of the page tables past the longest sequence's: a call goes by what its table allows, so that with many of
    them even short sequences are cut into tiles and shares"""
    global EXTRA
    EXTRA = request.param


def run_chunk(lib, c, q, qk, n, lens, window, n_heads, scale, m=None, out_stride=None):
    """rows of the type's bits -> (out bits, out as float32); out starts as 0x3F3F..."""
    m = m or len(q)
    os = out_stride or n_heads * c.hd
    out = filled(lib, m * os * q.dtype.itemsize, 0x3F)
    dq, cu, dl = dbuf(lib, q), dbuf(lib, pn.starts(n)), dbuf(lib, np.asarray(lens, np.int32))
    part = filled(lib, lib.L.g4_attn_chunk_paged_part_bytes(m, n_heads, c.n_kv, c.hd))
    lib.g4_attn_chunk_paged(dq.ptr, q.shape[1], qk, *c.args(), cu.ptr, dl.ptr, len(n), m, window, n_heads, F(scale), part.ptr,
                            out.ptr, os)
    lib.g4_sync()
    bits = out.to_array(NPT[qk]).reshape(m, os)
    return bits, (pn.bf16_back(bits) if qk == pn.BF16 else bits.astype(np.float32))


def bound_of(bound, want, q, k, v, qk, ck, scale):
    """what the operands' roundings add to the bound of fp32 arithmetic; q [rows, heads, hd], k, v [keys, kv, hd]"""
    big = np.abs(v).max()
    if qk != pn.F32:
        # weights rounded to the type once (each off by HALF of itself: of sum p |v|, which is at most max |v|, and by the
        # smallest subnormal's half at a maximum of 1) and the result rounded to it
        return bound + pn.HALF[qk] * (np.abs(want) + 1.01 * big) + 2.0 ** -25 * len(k) * big
    if ck in (pn.BF16, pn.Q8):
        return bound + 2.0 ** -23 * big         # weights as three bf16 terms, themselves; times a scale of codes: 2^-24
    # operands within 2^-22 of themselves or 2^-39 of their row's largest (F32: q and K, and the smaller terms' product
    # left out): a score is off by that of sum |q| |k|, its weight by twice it; weights and V 2^-22 each
    kv = np.repeat(np.abs(k), q.shape[1] // k.shape[1], 1)
    mags = np.abs(scale) * np.einsum("rhd,khd->rhk", np.abs(q), kv, optimize=True).max(-1)[..., None]
    low = np.abs(scale) * 2.0 ** -39 * k.shape[-1] * np.abs(q).max(-1, keepdims=True) * np.abs(k).max()
    each = 3 if ck == pn.F32 else 1
    return bound + each * (2 * (2.0 ** -22 * mags + 2 * low) + 2.0 ** -22 + 2.0 ** -39) * big


def check(lib, seed, combo, hd, n_heads, n_kv, page, n, hist, window=0, scale=None, gain=2.0, pad=0, extra=0, some=None):
    qk, ck = combo
    rng = np.random.default_rng(seed)
    scale = hd ** -0.5 if scale is None else scale
    lens = [a + b for a, b in zip(n, hist)]
    c = Cache(lib, rng, ck, hd, n_kv, page, lens, extra=EXTRA)
    k, v = rows(rng, sum(lens), n_kv, hd), rows(rng, sum(lens), n_kv, hd)
    c.store(k, v, lens, lens)
    q, qf = cast(rows(rng, sum(n) + pad, 1, n_heads * hd + extra) * np.float32(gain), qk)
    bits, got = run_chunk(lib, c, q, qk, n, lens, window, n_heads, scale, out_stride=n_heads * hd + extra)
    hk, hv = (pn.held(x, ck, hd).reshape(-1, n_kv, hd) for x in (k, v))
    at, key = pn.starts(n), pn.starts(lens)
    for s, (t, h) in enumerate(zip(n, hist)):
        for lo in range(0, t, 64):
            hi = min(t, lo + 64)
            if some is not None and lo and hi < t and lo // 64 % some:
                continue
            last = h + hi
            first = [max(0, h + i + 1 - window) if window else 0 for i in range(lo, hi)]
            kk = slice(key[s] + first[0], key[s] + last)
            qq = qf[at[s] + lo:at[s] + hi, :n_heads * hd].reshape(hi - lo, n_heads, hd)
            want, bound = pn.attention(qq, hk[kk], hv[kk], np.array(first) - first[0], scale)
            bound = bound_of(bound, want, qq, hk[kk], hv[kk], qk, ck, scale)
            err = np.abs(got[at[s] + lo:at[s] + hi, :n_heads * hd].reshape(hi - lo, n_heads, hd) - want)
            within(err, bound, (s, lo))
    untouched = np.full(1, 0x3F3F3F3F, np.uint32).view(bits.dtype)[0]
    assert (bits[sum(n):] == untouched).all() and (bits[:, n_heads * hd:] == untouched).all()


N = [1, 0, 31, 33, 5, 70, 129, 2, 1]
HIST = [0, 7, 100, 0, 300, 64, 1, 511, 63]


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_types(lib, combo, hd):
    """every pair of types and head_dim; rows that begin a sequence, that go on, one alone, none; rows past the last"""
    check(lib, 300 + hd, combo, hd, 8, 2, 16, N, HIST, pad=5)


@pytest.mark.parametrize("n_heads,n_kv", [(1, 1), (3, 3), (5, 1), (8, 1), (10, 2), (12, 1), (24, 8), (20, 1), (40, 2), (70, 1),
                                          (150, 1), (300, 1)])
def test_heads(lib, n_heads, n_kv):
    """one head to hundreds on a kv head"""
    for combo, hd in ((COMBOS[0], 128), (COMBOS[5], 64), (COMBOS[3], 64)):
        check(lib, 320 + n_heads, combo, hd, n_heads, n_kv, 32, [9, 1, 40], [3, 130, 70])


@pytest.mark.parametrize("window", [1, 5, 32, 64, 100, 512])
@pytest.mark.parametrize("combo,hd,page", [(COMBOS[0], 256, 16), (COMBOS[1], 128, 32), (COMBOS[5], 512, 64), (COMBOS[6], 256, 16),
                                           (COMBOS[2], 512, 16)])
def test_window(lib, window, combo, hd, page):
    check(lib, 340 + window, combo, hd, 4, 2, page, [3, 96, 150, 1, 33], [0, 40, 700, 600, 31], window=window)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd,n,hist", [(64, [3], [20011]), (256, [200, 1, 7], [5000, 3000, 0]), (512, [40, 2], [2777, 9000])])
def test_long(lib, combo, hd, n, hist):
    """long histories, split over many workgroups"""
    check(lib, 360, combo, hd, 4, 2, 64, n, hist, some=3, gain=1.0)


@pytest.mark.parametrize("combo,hd,window", [(COMBOS[0], 256, 512), (COMBOS[0], 512, 0), (COMBOS[5], 256, 0), (COMBOS[4], 128, 300)])
def test_prompts(lib, combo, hd, window):
    """thousands of rows, first ones and later ones"""
    check(lib, 361, combo, hd, 4, 1, 32, [1500, 1777], [0, 1001], window=window, some=12)


def test_many(lib):
    """hundreds of sequences of a few rows, with some long ones among them; the most there may be"""
    rng = np.random.default_rng(362)
    n = [int(x) for x in rng.integers(0, 4, 700)]
    hist = [int(x) for x in rng.integers(0, 60, 700)]
    check(lib, 362, COMBOS[5], 64, 2, 1, 16, n, hist)
    n[5], hist[600], n[699] = 150, 4000, 1
    check(lib, 363, COMBOS[3], 64, 2, 1, 16, n[:65] + n[600:], hist[:65] + hist[600:])
    check(lib, 364, COMBOS[6], 64, 1, 1, 16, [int(x) for x in rng.integers(0, 3, 4096)], [int(x) for x in rng.integers(0, 20, 4096)])


def test_lengths(lib):
    """histories and rows on either side of blocks, tiles and shares of the work"""
    for i, h in enumerate([0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 255]):
        check(lib, 370 + i, COMBOS[5], 64, 4, 1, 16, [32, 33, 1, 16], [h, h + 1, 3 * h, 0], gain=1.0)
    for h in (32 * 256 - 1, 32 * 256, 32 * 257):
        check(lib, 371, COMBOS[5], 64, 1, 1, 64, [1], [h], gain=1.0)
        check(lib, 372, COMBOS[0], 64, 2, 1, 64, [1, 40], [h, 70], gain=1.0)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
def test_strides(lib, combo):
    check(lib, 380, combo, 128, 4, 2, 32, [50, 7], [3, 90], extra=8, pad=2)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
def test_extremes(lib, combo):
    """weights on one key, equal weights, a negative scale, none, magnitudes far from 1"""
    for n, hist in (([90], [60]), ([5], [900])):
        check(lib, 381, combo, 128, 4, 2, 16, n, hist, gain=60.0 if combo[0] == pn.F32 else 20.0, scale=1.0)
        check(lib, 382, combo, 128, 4, 2, 16, n, hist, gain=0.0, scale=1.0)
        check(lib, 383, combo, 128, 4, 2, 16, n, hist, scale=-0.09)
        check(lib, 384, combo, 128, 4, 2, 16, n, hist, scale=0.0)
        if combo[0] != pn.F16:
            check(lib, 385, combo, 128, 4, 2, 16, n, hist, gain=1e-18, scale=1e17)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
def test_next_to_no_scores(lib, combo):
    """rows of zeros and a scale so small that their product is below fp32's smallest number"""
    for n, hist in (([90], [60]), ([5], [900])):
        for gain in (0.0, 1e-30):
            for scale in (1e-9, 1e-38):
                check(lib, 386, combo, 128, 4, 2, 16, n, hist, gain=gain, scale=scale)
                check(lib, 387, combo, 512, 4, 2, 16, n, hist, gain=gain, scale=-scale)


def test_window_pages_gone(lib):
    """pages that no row sees have been given away: entries that are no page, or another sequence's with NaN in it"""
    rng = np.random.default_rng(390)
    hd, n_kv, page, t, w, new = 128, 1, 16, 200, 50, 20
    for combo in COMBOS:
        c = Cache(lib, rng, combo[1], hd, n_kv, page, [t], extra=EXTRA)
        k, v = rows(rng, t, n_kv, hd), rows(rng, t, n_kv, hd)
        c.store(k, v, [t], [t])
        q = cast(rows(rng, new, 2, hd), combo[0])[0]
        a, af = run_chunk(lib, c, q, combo[0], [new], [t], w, 2, 0.1)
        c.table[0, :(t - new + 1 - w) // page] = -1
        c.dtable = dbuf(lib, c.table)
        b, _ = run_chunk(lib, c, q, combo[0], [new], [t], w, 2, 0.1)
        assert np.isfinite(af).all() and same_bits(a, b)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_pages_outside(lib, combo, hd):
    """a page outside the pool: NaN in the rows that see it and nowhere else"""
    rng = np.random.default_rng(391)
    n, lens, w = [40, 40, 3], [90, 90, 90], 30
    c = Cache(lib, rng, combo[1], hd, 1, 16, lens, extra=EXTRA)
    x = rows(rng, 270, 1, hd)
    c.store(x, x, lens, lens)
    q = cast(rows(rng, 83, 2, hd), combo[0])[0]
    for window in (0, w):
        a, _ = run_chunk(lib, c, q, combo[0], n, lens, window, 2, 0.1)
        old = c.table.copy()
        c.table[1, 4], c.table[2, 0] = c.pages, -5            # positions 64 .. 79; 0 .. 15
        c.dtable.write(c.table)
        b, bf = run_chunk(lib, c, q, combo[0], n, lens, window, 2, 0.1)
        c.table = old
        c.dtable.write(old)
        assert same_bits(a[:40], b[:40])
        p = np.arange(50, 90)
        sees = (p >= 64) & (p - window + 1 <= 79 if window else True)
        assert np.isnan(bf[40:80][sees]).all() and same_bits(a[40:80][~sees], b[40:80][~sees])
        if window:
            assert same_bits(a[80:], b[80:])
        else:
            assert np.isnan(bf[80:]).all()


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("combo", COMBOS, ids=str)
def test_not_finite(lib, combo, hd):
    """infinities and NaN in later rows, before the window, in other heads and other sequences change no row that does not
    see them; rows that see them are what the formula gives or NaN there"""
    rng = np.random.default_rng(392)
    n_kv, n_heads, n, hist, w = 2, 4, [70, 50], [60, 20], 40
    lens = [130, 70]
    c = Cache(lib, rng, combo[1], hd, n_kv, 16, lens, extra=EXTRA)
    k, v = rows(rng, 200, n_kv, hd), rows(rng, 200, n_kv, hd)
    c.store(k, v, lens, lens)
    q = cast(rows(rng, 120, n_heads, hd), combo[0])[0]
    for window in (0, w):
        a, _ = run_chunk(lib, c, q, combo[0], n, lens, window, n_heads, 0.1)
        k2, v2 = k.copy(), v.copy()
        v2[100, hd + 3] = np.inf        # sequence 0, position 100, kv head 1
        k2[110, 5] = NAN                # position 110, kv head 0
        v2[8, 7] = -np.inf              # position 8, kv head 0
        c.store(k2, v2, lens, lens)
        b, bf = run_chunk(lib, c, q, combo[0], n, lens, window, n_heads, 0.1)
        c.store(k, v, lens, lens)
        a4, b4, f4 = (x.reshape(120, n_heads, hd) for x in (a, b, bf))
        p = np.arange(60, 130)
        sees1 = (p >= 100) & ((p - w + 1 <= 100) | (window == 0))
        sees0 = ((p >= 110) & ((p - w + 1 <= 110) | (window == 0))) | (window == 0)
        assert same_bits(a4[70:], b4[70:])
        assert same_bits(a4[:70][~sees1, 2:], b4[:70][~sees1, 2:]) and not np.isfinite(f4[:70][sees1, 2:, 3]).any()
        assert same_bits(a4[:70][~sees0, :2], b4[:70][~sees0, :2]) and not np.isfinite(f4[:70][sees0, :2, 7]).any()


def test_misfits_are_left(lib):
    """more rows than positions, past the table, past the rows: those rows stay as they are, the others are done"""
    rng = np.random.default_rng(393)
    hd = 64
    c = Cache(lib, rng, pn.F32, hd, 1, 16, [40] * 4, extra=0)       # 48 positions each
    x = rows(rng, 160, 1, hd)
    c.store(x, x, [40] * 4, [40] * 4)
    q = rows(rng, 24, 2, hd)
    good, _ = run_chunk(lib, c, q, pn.F32, [6, 6, 6, 6], [40] * 4, 0, 2, 0.1)
    got, gf = run_chunk(lib, c, q, pn.F32, [6, 6, 6, 6], [40, 5, 49, 40], 0, 2, 0.1)
    assert same_bits(got[:6], good[:6]) and same_bits(got[18:], good[18:])
    assert (got[6:18].view(np.uint32) == 0x3F3F3F3F).all()
    out = filled(lib, 24 * 2 * hd * 4, 0x3F)
    dq, dl = dbuf(lib, q), dbuf(lib, np.array([40] * 4, np.int32))
    part = filled(lib, lib.L.g4_attn_chunk_paged_part_bytes(24, 2, 1, hd))
    for cu in ([0, 6, 5, -3, 200], [0, 6, 12, 30, 24], [-7, -1, 3, 2, 1 << 30]):
        dcu = dbuf(lib, np.array(cu, np.int32))
        lib.g4_memset(out.ptr, 0x3F, out.nbytes)
        lib.g4_attn_chunk_paged(dq.ptr, 2 * hd, pn.F32, *c.args(), dcu.ptr, dl.ptr, 4, 24, 0, 2, F(0.1), part.ptr, out.ptr, 2 * hd)
        lib.g4_sync()
        o = out.to_array(np.uint32).reshape(24, -1)
        ok = [s for s in range(4) if 0 <= cu[s] < cu[s + 1] <= 24]
        may = np.zeros(24, bool)
        for s in ok:
            may[cu[s]:cu[s + 1]] = True
        assert (o[~may] == 0x3F3F3F3F).all()


@pytest.mark.parametrize("combo,hd", [(COMBOS[0], 256), (COMBOS[5], 512), (COMBOS[3], 64), (COMBOS[6], 256)])
def test_captured(lib, combo, hd):
    """captured once, replayed with other lengths and rows, the program's own eager work and another captured call that
    shares the scratch in between: each replay is the eager call, bit for bit"""
    rng = np.random.default_rng(394)
    heads, kv, page, m = 8, 2, 16, 160
    qk, ck = combo
    plans = [([100, 1, 30], [20, 900, 0]), ([1, 1, 1], [120, 901, 30]), ([0, 150, 3], [121, 0, 1000]), ([53, 53, 54], [300, 40, 0])]
    total = [max(p[0][s] + p[1][s] for p in plans) for s in range(3)]
    with Stream(lib):
        c = Cache(lib, rng, ck, hd, kv, page, total, extra=EXTRA)
        x = rows(rng, sum(total), kv, hd)
        c.store(x, x[::-1].copy(), total, total)
        q = [cast(rows(rng, m, heads, hd), qk)[0] for _ in plans]
        dq, cu, dl = dbuf(lib, q[0]), dbuf(lib, np.zeros(4, np.int32)), dbuf(lib, np.zeros(3, np.int32))
        outs = [filled(lib, q[0].nbytes, 0x3F) for _ in range(3)]
        part = filled(lib, lib.L.g4_attn_chunk_paged_part_bytes(m, heads, kv, hd))

        def call(out, window):
            lib.g4_attn_chunk_paged(dq.ptr, heads * hd, qk, *c.args(), cu.ptr, dl.ptr, 3, m, window, heads, F(0.1), part.ptr,
                                    out.ptr, heads * hd)

        graphs = []
        for out, window in ((outs[0], 0), (outs[1], 60)):
            lib.g4_graph_begin()
            call(out, window)
            g = C.c_void_p()
            lib.g4_graph_end(C.byref(g))
            graphs.append(g.value)
        for again in range(2):
            for (n, hist), qi in zip(plans, q):
                dq.write(qi)
                cu.write(pn.starts(n))
                dl.write(np.add(n, hist).astype(np.int32))
                for i, window in ((0, 0), (1, 60)):
                    lib.g4_memset(outs[i].ptr, 0x3F, outs[i].nbytes)
                    lib.g4_memset(outs[2].ptr, 0x3F, outs[2].nbytes)
                    lib.g4_graph_launch(graphs[0])
                    lib.g4_graph_launch(graphs[1])
                    call(outs[2], window)
                    lib.g4_sync()
                    assert same_bits(outs[i].to_array(np.uint8), outs[2].to_array(np.uint8)), (again, n, i)
        for g in graphs:
            lib.g4_graph_destroy(g)


@pytest.mark.parametrize("combo", [COMBOS[0], COMBOS[4], COMBOS[6]], ids=str)
def test_offsets_past_32_bits(lib, combo):
    """pages at the end of pools of more than 4 GB"""
    rng = np.random.default_rng(395)
    hd, n_kv, page, n, lens = 512, 2, 64, [40, 3], [200, 90]
    per = lib.L.g4_kv_pool_bytes(combo[1], 1, page, n_kv, hd)
    pages = (5 << 30) // per
    need = [4, 2]
    table = np.full((2, 5), -1, np.int32)
    table[0, :4], table[1, :2] = pages - 1 - np.arange(4), [pages - 5, pages // 2]
    c = Cache(lib, rng, combo[1], hd, n_kv, page, None, table=table, pages=pages)
    k, v = rows(rng, 290, n_kv, hd), rows(rng, 290, n_kv, hd)
    c.store(k, v, lens, lens)
    q = cast(rows(rng, 43, 4, hd), combo[0])[0]
    big, _ = run_chunk(lib, c, q, combo[0], n, lens, 0, 4, 0.05)
    small = Cache(lib, rng, combo[1], hd, n_kv, page, lens, extra=EXTRA)
    small.store(k, v, lens, lens)
    assert sum(need) <= small.pages
    assert same_bits(big, run_chunk(lib, small, q, combo[0], n, lens, 0, 4, 0.05)[0])


def test_shared_pages(lib):
    """two sequences with the same first pages (a common prefix) and rows of their own: each what it would be alone"""
    rng = np.random.default_rng(396)
    hd, page = 128, 16
    for combo in COMBOS:
        table = np.array([[0, 1, 2, 3, 4], [0, 1, 2, 5, 6]], np.int32)
        c = Cache(lib, rng, combo[1], hd, 1, page, None, table=table, pages=7)
        x = rows(rng, 48 + 20 + 27, 1, hd)
        c.store(x[:48], x[:48], [48, 0], [48, 48])
        c.store(x[48:], x[48:], [20, 27], [68, 75])
        q = cast(rows(rng, 47, 2, hd), combo[0])[0]
        both, _ = run_chunk(lib, c, q, combo[0], [20, 27], [68, 75], 0, 2, 0.1)
        want = []
        for i, (r0, r1) in enumerate(((0, 20), (20, 47))):
            f = pn.held(np.concatenate([x[:48], x[48 + r0:48 + r1]]), combo[1], hd).reshape(-1, 1, hd)
            qf = pn.bf16_back(q[r0:r1]) if combo[0] == pn.BF16 else q[r0:r1].astype(np.float32)
            o, b = pn.attention(qf.reshape(-1, 2, hd), f, f, [0] * (r1 - r0), 0.1)
            want.append((o, bound_of(b, o, qf.reshape(-1, 2, hd), f, f, *combo, 0.1)))
        gf = pn.bf16_back(both) if combo[0] == pn.BF16 else both.astype(np.float32)
        for (r0, r1), (o, b) in zip(((0, 20), (20, 47)), want):
            within(np.abs(gf[r0:r1].reshape(-1, 2, hd) - o), b, combo)


@pytest.mark.parametrize("combo,hd,window", [(COMBOS[0], 256, 100), (COMBOS[5], 256, 100), (COMBOS[3], 512, 0), (COMBOS[6], 512, 0)])
def test_serving(lib, combo, hd, window):
    """The operators as a server uses them, from raw projections: prompts in pieces and later turns beside single tokens,
    each step one append (norms, rotation, pages) and one attention over the cache.  Every output is the formula's of the
    whole sequences in 64 bits, with the rows as the append left them."""
    rng = np.random.default_rng(397)
    qk, ck = combo
    heads, kv, page, scale = 8, 2, 16, 1.0
    steps = [[37, 0, 1], [60, 5, 1], [1, 30, 1], [1, 1, 1], [0, 8, 40]]
    total = np.sum(steps, 0)
    from test_gpu_qkv_seqs import Rows
    c = Cache(lib, rng, ck, hd, kv, page, [int(t) for t in total], extra=EXTRA)
    outs, qs = [[[] for _ in range(3)] for _ in range(2)]
    had = np.zeros(3, int)
    kw = None
    for n in steps:
        had = had + n
        r = Rows(lib, np.random.default_rng(int(had.sum())), n, [int(x) for x in had], heads, kv, hd, hd, wide=0)
        if kw is None:
            kw = r.w[1] * np.float32(hd ** -0.5)
        r.d[4].write(kw)
        size = 4 if qk == pn.F32 else 2
        qo = filled(lib, r.m * heads * hd * size)
        lib.g4_kv_page_append(*c.args(), *r.kv_in(), *r.q_in(), qo.ptr, heads * hd, qk, *r.turn(), *r.seqs())
        q = qo.to_array(NPT[qk]).reshape(r.m, -1)
        o = run_chunk(lib, c, q, qk, n, had, window, heads, scale)[1]
        qf = pn.bf16_back(q) if qk == pn.BF16 else q
        for s, (a, b) in enumerate(zip(pn.starts(n)[:-1], pn.starts(n)[1:])):
            outs[s].append(o[a:b])
            qs[s].append(qf[a:b])
    total = [int(t) for t in total]
    gk, gv = c.load(total, total)
    at = pn.starts(total)
    assert np.isfinite(gk).all() and np.isfinite(gv).all()
    for s, t in enumerate(total):
        k, v = (x[at[s]:at[s + 1]].reshape(t, kv, hd) for x in (gk, gv))
        q, o = (np.concatenate(x[s]).reshape(t, heads, hd) for x in (qs, outs))
        first = [max(0, i + 1 - window) if window else 0 for i in range(t)]
        want, bound = pn.attention(q, k, v, first, scale)
        within(np.abs(o - want), bound_of(bound, want, q, k, v, qk, ck, scale), s)


def check_far(lib, hd, k, v, gain, window=0, seed=380):
    """fp32 rows over fp32 keys whose sizes differ much from key to key: the last 70 positions of one sequence"""
    rng = np.random.default_rng(seed)
    t, n, n_heads, n_kv, scale = len(v), 70, 8, 2, hd ** -0.5
    c = Cache(lib, rng, pn.F32, hd, n_kv, 16, [t], extra=EXTRA)
    c.store(k, v, [t], [t])
    q = rows(rng, n, n_heads, hd) * np.float32(gain)
    _, got = run_chunk(lib, c, q, pn.F32, [n], [t], window, n_heads, scale)
    first = [max(0, t - n + i + 1 - window) if window else 0 for i in range(n)]
    q, k, v = (x.reshape(len(x), -1, hd) for x in (q, k, v))
    want, bound = pn.attention(q, k, v, first, scale)
    big = np.abs(v).max(-1).repeat(n_heads // n_kv, 1).astype(np.float64)
    for i in range(n):
        seen = slice(first[i], t - n + i + 1)
        for h in range(n_heads):
            kh, vh = k[seen, h // (n_heads // n_kv)].astype(np.float64), np.abs(v[seen, h // (n_heads // n_kv)])
            p = scale * (kh @ q[i, h])
            p = np.exp(p - p.max())
            pb = p * big[seen, h]
            # An element of V is met within 2^-39 of its row's largest; a weight times its V row's power of two is held
            # as two fp16, the largest of them at 2^11 or more and each within 2^-25: times V's scaled elements, below
            # 2^15, that is 2^-10 a key where the largest stands for 2^11 * 2^14 at least, 2^-35 of it.
            bound[i, h] += (2.0 ** -38 * pb.sum() + 2.0 ** -35 * len(p) * pb.max()) / p.sum()
            # Rows of V below 2^-76 have the scale of 2^-76, 2^90: halves within 2^-25 of the scaled row are 2^-115 of V.
            bound[i, h] += 2.0 ** -115
            # A score has the row's exponent (-90 to 113) added and the maximum taken off: two roundings of numbers
            # below 256, 2^-17 each and times ln 2 in a weight, met in the numerator and in the denominator.
            bound[i, h] += 4 * np.log(2) * 2.0 ** -17 * (p @ vh) / p.sum()
    within(np.abs(got.reshape(n, n_heads, hd) - want), bound, hd)


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("top", [61, 62, 100, 117])
@pytest.mark.parametrize("big_first", [False, True])
def test_values_far_apart(lib, hd, top, big_first):
    """V rows of zeros beside one of 2^61 and more, in front of it and behind it, with equal scores and with scores far
    apart: a row of zeros takes its share of the weights whatever the others hold"""
    rng = np.random.default_rng(381)
    t = 150
    k, v = rows(rng, t, 2, hd), np.zeros((t, 2 * hd), np.float32)
    v[3 if big_first else 77] = np.float32(1.5 * 2.0 ** top)
    check_far(lib, hd, k, v, 0.0)
    check_far(lib, hd, k, v, 6.0)
    # tiny rows, in tiles of their own and beside large ones, and a window
    v = rows(rng, t, 2, hd) * np.exp2(np.where(np.arange(t) // 40 % 2 == big_first, top - 3, -103)).astype(np.float32)[:, None]
    v[rng.integers(0, t, 9)] = 0
    check_far(lib, hd, k, v, 3.0)
    for window in (70, 270):
        check_far(lib, hd, np.concatenate([k] * 3), np.concatenate([v] * 3), 3.0, window=window)


@pytest.mark.parametrize("hd,window", [(64, 40), (64, 260), (256, 0), (256, 130), (512, 0), (512, 70)])
def test_magnitudes(lib, hd, window):
    """fp32 rows whose sizes differ by 2^60 from key to key and by 2^20 within a row: what a row does not see, and what
    has next to no weight, costs it no precision, and a key of large scores moves the maximum far at once"""
    rng = np.random.default_rng(390 + hd)
    t = 430
    k, v = rows(rng, t, 2, hd), rows(rng, t, 2, hd)
    v *= np.exp2(rng.integers(-30, 31, (t, 2 * hd // 64))).repeat(64, 1).astype(np.float32)
    v *= np.exp2(rng.integers(-10, 11, v.shape)).astype(np.float32)
    k *= np.exp2(rng.integers(-6, 3, (t, 1))).astype(np.float32)
    k[rng.integers(0, t, 12)] *= np.float32(20)
    v[7] = v[200] = k[31] = 0
    check_far(lib, hd, k, v, 1.0, window=window)


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("combo", [COMBOS[2], COMBOS[3], COMBOS[5], COMBOS[6]], ids=str)
def test_values_at_the_limit(lib, combo, hd):
    """V so large that the keys together stay just below fp32's largest number, under scores that rise by 2^7.9 from one
    pair of tiles to the next"""
    qk, ck = combo
    t, n, n_heads, n_kv, top = 400, 70, 8, 2, 119
    assert t * 2.0 ** top < float(np.finfo(np.float32).max) < t * 2.0 ** (top + 1)
    rng = np.random.default_rng(394)
    k = np.zeros((t, n_kv, hd), np.float32)
    for i in range(t):
        k[i, :, :i // 64] = 1
    v = np.full((t, n_kv * hd), 2.0 ** top, np.float32)
    v *= rng.choice(np.array([1, -1], np.float32), n_kv * hd)
    q = np.zeros((n, n_heads, hd), np.float32)
    q[:, :, :16] = 5.46875
    c = Cache(lib, rng, ck, hd, n_kv, 16, [t], extra=EXTRA)
    c.store(k.reshape(t, -1), v, [t], [t])
    _, got = run_chunk(lib, c, cast(q.reshape(n, -1), qk)[0], qk, [n], [t], 0, n_heads, 1.0)
    hk, hv = (pn.held(x.reshape(t, -1), ck, hd).reshape(t, n_kv, hd) for x in (k, v))
    want, bound = pn.attention(q, hk, hv, [0] * n, 1.0)
    within(np.abs(got.reshape(n, n_heads, hd) - want), bound_of(bound, want, q, hk, hv, qk, ck, 1.0), hd)


FIRST = """
import ctypes as C, sys
import numpy as np
sys.path[:0] = {paths!r}
import g4, paged_np as pn, test_gpu_paged as base
lib = g4.Lib.get()
lib.init(0)
with base.Stream(lib):
    rng = np.random.default_rng(395)
    kind, hd, n_heads, n_kv, n, lens = {kind}, {hd}, 8, 2, [200, 100], [500, 100]
    c = base.Cache(lib, rng, kind, hd, n_kv, 16, lens, extra=2000)
    k, v = base.rows(rng, 600, n_kv, hd), base.rows(rng, 600, n_kv, hd)
    c.store(k, v, lens, lens)
    q = base.cast(base.rows(rng, 300, n_heads, hd), kind)[0]
    dq, cu, dl = base.dbuf(lib, q), base.dbuf(lib, pn.starts(n)), base.dbuf(lib, np.asarray(lens, np.int32))
    out = base.filled(lib, q.nbytes)
    part = base.filled(lib, lib.L.g4_attn_chunk_paged_part_bytes(300, n_heads, n_kv, hd))
    call = lambda: lib.g4_attn_chunk_paged(dq.ptr, n_heads * hd, kind, *c.args(), cu.ptr, dl.ptr, 2, 300, 0, n_heads,
                                           C.c_float(0.1), part.ptr, out.ptr, n_heads * hd)
    lib.g4_graph_begin()
    call()
    g = C.c_void_p()
    lib.g4_graph_end(C.byref(g))
    got = []
    for i in range(4):
        lib.g4_memset(out.ptr, 0x3F, out.nbytes)
        if i == 2:
            call()
        else:
            lib.g4_graph_launch(g.value)
        lib.g4_sync()
        got.append(out.to_array(np.uint8))
    lib.g4_graph_destroy(g.value)
    assert all(np.array_equal(a, got[2]) for a in got)
    assert (got[0].reshape(300, -1) != 0x3F).any(1).all()
print("FIRST OK")
"""


def test_first_call_captured():
    """a process whose first call of the operator is a captured one (kernels with more than 64 KB of LDS)"""
    if EXTRA != 2:
        return
    here = os.path.dirname(os.path.abspath(__file__))
    paths = [here, os.path.join(os.path.dirname(here), "gemma4.c_amd")]
    for kind, hd in ((pn.F32, 512), (pn.BF16, 256)):
        r = subprocess.run([sys.executable, "-c", FIRST.format(paths=paths, kind=kind, hd=hd)], capture_output=True, text=True,
                           timeout=100)
        assert r.returncode == 0 and "FIRST OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
