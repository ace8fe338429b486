"""Attention of chunks of new rows over the paged cache where the call is cut
into tiles and shares of them (g4_attn_chunk_paged), against the formula in 64
bits.  A call of few keys takes another kernel, by the keys that its window or
its table allows and by its rows: here each case says which of the two it is for
and is checked to be one that goes there."""
import ctypes as C

import numpy as np
import pytest

import paged_np as pn
import test_gpu_chunk as tc
from test_gpu_chunk import COMBOS, bound_of, run_chunk
from test_gpu_paged import NAN, NPT, Cache, cast, dbuf, filled, rows, same_bits, within

pytestmark = pytest.mark.gpu

F = C.c_float
SIZE = {pn.F32: 4, pn.F16: 2, pn.BF16: 2, pn.Q8: 1}
WIDE = 3000     # entries of a table past the longest sequence's


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


def tiles(c, window, m, n_heads):
    """whether a call of m rows over cache c goes to the tiles: more than 256 keys a row, as its window or table allows, in
    units of 512 bytes of a key's row, or 2^17 of them over all rows and heads"""
    keys = c.table.shape[1] * c.page
    keys = min(keys, window) if window else keys
    keys *= max(1, c.hd * SIZE[c.kind] // 512)
    return keys > 256 or keys * m * n_heads > 1 << 17


def rows_for_tiles(c, window, n_heads):
    """a number of rows (used or not) with which a call goes to the tiles whatever its window"""
    return ((1 << 17) // (min(window, c.table.shape[1] * c.page) * n_heads) + 1) if window else 1


def padded(q, m):
    """q with rows that belong to no sequence behind it, m in all: ones, and NaN in a few of them"""
    x = np.ones((max(m, len(q)), q.shape[1]), np.float32).astype(q.dtype) if q.dtype != np.uint16 else np.full(
        (max(m, len(q)), q.shape[1]), 0x3F80, np.uint16)
    x[:len(q)] = q
    if len(x) > len(q):
        x[-1] = np.full(1, NAN).astype(q.dtype)[0] if q.dtype != np.uint16 else 0x7FC0
    return x


def back(bits, kind):
    return pn.bf16_back(bits) if kind == pn.BF16 else bits.astype(np.float32)


def store_prefix(c, k, v):
    """rows into the pages of the table's first sequence"""
    c.store(k, v, [len(k)] + [0] * (len(c.table) - 1), [len(k)] * len(c.table))


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("gain", [[1.0], [1.0, 0.9, 0.8, 0.75], [1.0, 0.5, 0.25, -1.0]], ids=["one", "alike", "apart"])
def test_scores_rise_far(lib, combo, hd, gain):
    """One row each of many sequences that share their pages, under scores that rise by 150 (216 in the exponent of 2) from
    64 keys to the next, in many places of many shares: what was summed before is of no weight, all of it, and is gone."""
    qk, ck = combo
    n_heads = len(gain)
    rng = np.random.default_rng(500 + hd)
    seqs, page, long = 120, 64, 640
    table = np.tile(np.concatenate([np.arange(long // page), np.full(WIDE, -1)]).astype(np.int32), (seqs, 1))
    c = Cache(lib, rng, ck, hd, 1, page, None, table=table, pages=long // page)
    assert tiles(c, 0, seqs, n_heads)
    step = 150.0 / hd
    k = np.repeat((np.arange(long) // 64 - 4) * step, hd).reshape(long, hd).astype(np.float32)
    v = rows(rng, long, 1, hd) + np.float32(1)
    store_prefix(c, k, v)
    hk, hv = (pn.held(x, ck, hd).reshape(long, 1, hd) for x in (k, v))
    lens = [int(x) for x in rng.integers(300, long + 1, seqs)]
    # a third of the sequences under smaller steps
    q = np.repeat(np.array(gain)[None] * np.where(np.arange(seqs) % 3, 1.0, 0.75)[:, None], hd, 1).astype(np.float32)
    q, qf = cast(q, qk)
    _, got = run_chunk(lib, c, q, qk, [1] * seqs, lens, 0, n_heads, 1.0)
    for s in range(seqs):
        qq = qf[s:s + 1].reshape(1, n_heads, hd)
        want, bound = pn.attention(qq, hk[:lens[s]], hv[:lens[s]], [0], 1.0)
        bound = bound_of(bound, want, qq, hk[:lens[s]], hv[:lens[s]], qk, ck, 1.0)
        within(np.abs(got[s].reshape(1, n_heads, hd) - want), bound, (s, lens[s]))


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("k_top,q_top", [(112, -110), (104, -100), (120, -120), (-110, 112), (-120, 120)])
@pytest.mark.parametrize("sign", [False, True])
def test_large_beside_small(lib, hd, k_top, q_top, sign):
    """fp32 rows over fp32: keys as large as fp32 has them beside rows so small that the scores are ordinary, and the other
    way round; keys of either sign, and of one"""
    rng = np.random.default_rng(510 + hd)
    n, lens, n_heads, n_kv = [70, 1], [300, 90], 4, 2
    c = Cache(lib, rng, pn.F32, hd, n_kv, 16, lens, extra=WIDE)
    assert tiles(c, 0, sum(n), n_heads)
    k, v = rows(rng, sum(lens), n_kv, hd), rows(rng, sum(lens), n_kv, hd)
    q = rows(rng, sum(n), n_heads, hd)
    if sign:
        k, q = np.abs(k), np.abs(q) * rng.choice(np.array([1, -1], np.float32), q.shape[1] // hd).repeat(hd)
    # scores stay ordinary: up to 4 hd a product of ones
    k, q = k * np.float32(2.0 ** k_top), (q * np.float32(2.0 ** q_top)).astype(np.float32)
    scale = (0.25 if not sign else 4 / hd) * 2.0 ** -(k_top + q_top)
    c.store(k, v, lens, lens)
    _, got = run_chunk(lib, c, q, pn.F32, n, lens, 0, n_heads, scale)
    at, key = pn.starts(n), pn.starts(lens)
    for s in range(2):
        kk = slice(key[s], key[s + 1])
        qq = q[at[s]:at[s + 1]].reshape(n[s], n_heads, hd).astype(np.float64)
        kf, vf = (x[kk].reshape(-1, n_kv, hd).astype(np.float64) for x in (k, v))
        want, bound = pn.attention(qq, kf, vf, [0] * n[s], scale)
        bound = bound_of(bound, want, qq, kf, vf, pn.F32, pn.F32, scale)
        within(np.abs(got[at[s]:at[s + 1]].reshape(n[s], n_heads, hd) - want), bound, s)


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("k_top,q_top", [(125, 125), (125, -100), (-100, 125)])
def test_rows_and_keys_that_do_not_meet(lib, hd, k_top, q_top):
    """fp32 rows over fp32 whose dims are zeros wherever the keys' are not: scores of 0, however large both are"""
    rng = np.random.default_rng(520 + hd)
    n, t, n_heads = 50, 200, 2
    c = Cache(lib, rng, pn.F32, hd, 1, 16, [t], extra=WIDE)
    assert tiles(c, 0, n, n_heads)
    k, v, q = rows(rng, t, 1, hd), rows(rng, t, 1, hd), rows(rng, n, n_heads, hd).reshape(n, n_heads, hd)
    on = rng.random(hd) < 0.5
    k, q = np.where(on, k, 0) * np.float32(2.0 ** k_top), np.where(on, 0, q) * np.float32(2.0 ** q_top)
    c.store(k.astype(np.float32), v, [t], [t])
    _, got = run_chunk(lib, c, q.reshape(n, -1).astype(np.float32), pn.F32, [n], [t], 0, n_heads, 1.0)
    zq, kf, vf = np.zeros((n, n_heads, hd)), np.zeros((t, 1, hd)), v.reshape(t, 1, hd).astype(np.float64)
    want, bound = pn.attention(zq, kf, vf, [0] * n, 1.0)
    within(np.abs(got.reshape(n, n_heads, hd) - want), bound_of(bound, want, zq, kf, vf, pn.F32, pn.F32, 1.0), hd)


# (log2 of q, of K, of the scale): q k leaves fp32's range, or comes near it, where scores do not
FAR = {pn.BF16: [(75, 50, -122), (5, 120, -122), (122, 3, -122), (122, 0, -120), (30, 90, -118), (-8, 122, -114), (-60, 120, -60),
                 (10, 10, -20)],
       pn.Q8: [(121, -2, -119), (117, 2, -119), (121, -20, -101), (60, 60, -120), (-30, 115, -85), (-100, 40, 60), (10, 10, -20)]}


@pytest.mark.parametrize("ck,case", [(ck, case) for ck in FAR for case in FAR[ck]], ids=str)
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("extra", [0, WIDE], ids=["table", "wide"])
def test_large_rows_under_a_small_scale(lib, ck, case, hd, extra):
    """bf16 rows whose products with the keys are far larger than the scores, which the scale makes ordinary; scales of
    either sign that are no power of two; some rows of zeros and far smaller rows among them.  The call of few keys and
    that of tiles agree with the formula."""
    rng = np.random.default_rng(530 + hd)
    n, lens, n_heads, n_kv = [70, 1, 9], [124, 90, 100], 4, 2
    c = Cache(lib, rng, ck, hd, n_kv, 16, lens, extra=extra)
    if extra:
        assert tiles(c, 0, sum(n), n_heads)
    k, v = rows(rng, sum(lens), n_kv, hd), rows(rng, sum(lens), n_kv, hd)
    q = rows(rng, sum(n), n_heads, hd)
    q[3], q[5], q[7] = 0, q[5] * 2.0 ** -4, q[7] * 2.0 ** -60
    k = (k * 2.0 ** case[1]).astype(np.float32)
    q, qf = cast((q * 2.0 ** case[0]).astype(np.float32), pn.BF16)
    c.store(k, v, lens, lens)
    hk, hv = (pn.held(x, ck, hd).reshape(-1, n_kv, hd).astype(np.float64) for x in (k, v))
    at, key = pn.starts(n), pn.starts(lens)
    for sign in (0.17, -0.23):
        scale = float(np.float32(sign * 2.0 ** case[2]))
        _, got = run_chunk(lib, c, q, pn.BF16, n, lens, 0, n_heads, scale)
        for s in range(len(n)):
            kk = slice(key[s], key[s + 1])
            qq = qf[at[s]:at[s + 1]].reshape(n[s], n_heads, hd).astype(np.float64)
            want, bound = pn.attention(qq, hk[kk], hv[kk], [0] * n[s], scale)
            bound = bound_of(bound, want, qq, hk[kk], hv[kk], pn.BF16, ck, scale)
            # q times the scale's power of two as bf16: half a step of its smallest, 2^-134, below its normal range; the rest
            # of the scale is below 2; a score's error twice, in the numerator and in the denominator
            bound = bound + 2 * 2 * 2.0 ** -134 * np.abs(hk[kk]).sum(-1).max() * np.abs(hv[kk]).max()
            within(np.abs(got[at[s]:at[s + 1]].reshape(n[s], n_heads, hd) - want), bound, (s, sign))


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("window", [0, 300])
def test_what_other_rows_see(lib, combo, hd, window):
    """keys behind a row and before its window, and the other rows and heads of its sequence: whatever they are, finite and
    large, tiny, infinite or NaN, the row is the formula's of what it sees, within the bound that it has without them"""
    qk, ck = combo
    rng = np.random.default_rng(540 + hd)
    n, t, n_heads, n_kv = 90, 420, 4, 2
    c = Cache(lib, rng, ck, hd, n_kv, 16, [t], extra=WIDE)
    assert tiles(c, window, n, n_heads)
    k, v = rows(rng, t, n_kv, hd), rows(rng, t, n_kv, hd)
    x = rows(rng, n, n_heads, hd)
    q, qf = cast(x, qk)
    scale = 2 * hd ** -0.5
    pos = np.arange(t - n, t)
    late, early = t - 30, 60                  # changed: late and behind it; with a window, up to early
    keep = pos < late
    if window:
        keep &= pos - window + 1 > early
    assert 20 < keep.sum() < n
    cut = np.arange(t) >= late
    if window:
        cut |= np.arange(t) <= early
    hk, hv = (pn.held(y, ck, hd).reshape(t, n_kv, hd) for y in (k, v))
    first = np.maximum(pos + 1 - window, 0) if window else pos * 0
    at = np.flatnonzero(keep)
    one, last = first[at[0]], pos[at[-1]] + 1
    qq = qf.reshape(n, n_heads, hd)[keep]
    want, bound = pn.attention(qq, hk[one:last], hv[one:last], first[keep] - one, scale)
    bound = bound_of(bound, want, qq, hk[one:last], hv[one:last], qk, ck, scale)

    def run(q):
        got = run_chunk(lib, c, q, qk, [n], [t], window, n_heads, scale)[1]
        return np.abs(got.reshape(n, n_heads, hd)[keep] - want)

    for what in ("nothing", "large", "rising", "tiny", "infinite", "minus infinite", "mixed"):
        k2, v2 = k.copy(), v.copy()
        if what == "large":
            k2[cut] *= 40
            v2[cut] *= 1000
        elif what == "rising":
            k2[cut] *= np.linspace(1, 5, cut.sum(), dtype=np.float32)[:, None]
        elif what == "tiny":
            k2[cut] = 0
            v2[cut] *= np.float32(2.0 ** -100) if ck != pn.F16 else np.float32(0)
        elif what == "infinite":
            k2[cut] = np.inf
            v2[cut] = -np.inf
        elif what == "minus infinite":
            k2[cut] = -np.inf
        elif what == "mixed":
            k2[late], k2[late + 3, 1], v2[late + 7, hd + 1], v2[late + 9] = NAN, np.inf, np.inf, NAN
            if window:
                k2[3, 5], v2[early, hd + 9], v2[20] = -np.inf, np.inf, np.inf
        c.store(k2, v2, [t], [t])
        within(run(q), bound, what)
    c.store(k, v, [t], [t])
    # another row's or head's q
    stay = np.arange(n)[keep] % 3 != 1
    for what in (8.0, 0.0, np.inf, NAN):
        y = x.reshape(n, n_heads, hd).copy()
        with np.errstate(all="ignore"):
            y[1::3] *= np.float32(what)
            y[:, 2] *= np.float32(what)
            err = run(cast(y.reshape(n, -1), qk)[0])
        within(err[stay][:, [0, 1, 3]], bound[stay][:, [0, 1, 3]], what)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd,window", [(64, 1), (64, 20), (128, 40), (256, 64), (64, 700), (256, 300), (512, 20), (512, 600)])
def test_last_positions_there_are(lib, combo, hd, window):
    """sequences that end at position 2^30 - 1, the last that a table allows: the same bits as at the end of a short sequence,
    by the tiles and by the call of few keys"""
    qk, ck = combo
    rng = np.random.default_rng(550 + hd)
    page, n, n_heads, n_kv = 4096, 50, 2, 1
    top, short = 1 << 30, 2 * page
    new = min(short, window + n + 3)
    k, v = rows(rng, new, n_kv, hd), rows(rng, new, n_kv, hd)
    q = cast(rows(rng, n, n_heads, hd), qk)[0]
    got = []
    for length in (short, top):
        width = (length + page - 1) // page
        table = np.full((1, width), -1, np.int32)
        table[0, -2:] = [1, 0]
        c = Cache(lib, rng, ck, hd, n_kv, page, None, table=table, pages=2)
        c.store(k, v, [new], [length])
        for m in (n, max(n, rows_for_tiles(c, window, n_heads))):
            if m > n:
                assert tiles(c, window, m, n_heads)
            bits, f = run_chunk(lib, c, padded(q, m), qk, [n], [length], window, n_heads, 0.1)
            assert np.isfinite(f[:n]).all()
            got.append(bits[:n])
    assert same_bits(got[0], got[2]) and same_bits(got[1], got[3])
    hk, hv = (pn.held(x, ck, hd).reshape(-1, n_kv, hd) for x in (k, v))
    qf = back(q, qk).reshape(n, n_heads, hd)
    first = [new - n + i + 1 - window for i in range(n)]
    want, bound = pn.attention(qf, hk, hv, first, 0.1)
    bound = bound_of(bound, want, qf, hk, hv, qk, ck, 0.1)
    for g in got[2:]:
        within(np.abs(back(g, qk).reshape(n, n_heads, hd) - want), bound, window)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("below", [20, 24, 26, 28])
def test_long_flat_tail(lib, hd, below):
    """fp16 rows: one key far above hundreds whose weights lie below fp16's own range beside it, and whose V is all there
    is.  A weight is within 2^-11 of itself or 2^-32 of the largest."""
    rng = np.random.default_rng(560 + hd)
    seqs, page, long = 300, 64, 1024
    table = np.tile(np.concatenate([np.arange(long // page), np.full(WIDE, -1)]).astype(np.int32), (seqs, 1))
    c = Cache(lib, rng, pn.F16, hd, 1, page, None, table=table, pages=long // page)
    assert tiles(c, 0, seqs, 1)
    k, v = np.zeros((long, hd), np.float32), 1000 + 100 * rows(rng, long, 1, hd)
    q = np.zeros((seqs, hd), np.float32)
    q[:, 0] = 1
    # the key that is above the others, at places all over the tiles
    tops = np.arange(5, long, 64)
    k[tops, 0] = np.round(below * np.log(2) * 16) / 16
    v[tops] = 0
    store_prefix(c, k, v)
    hk, hv = (pn.held(x, pn.F16, hd).reshape(long, 1, hd) for x in (k, v))
    lens = [int(x) for x in rng.integers(600, long + 1, seqs)]
    q, qf = cast(q, pn.F16)
    _, got = run_chunk(lib, c, q, pn.F16, [1] * seqs, lens, 0, 1, 1.0)
    for s in range(seqs):
        t = lens[s]
        want, bound = pn.attention(qf[s:s + 1].reshape(1, 1, hd), hk[:t], hv[:t], [0], 1.0)
        # the weights' rounding and the result's, each 2^-11 of the sum (V is positive); below fp16's normal range a weight
        # is off by half a step of 2^-24 where the largest is 2^7 at least, 2^-32 of it, and all of them are divided by a
        # sum of `above` such largest ones; the result's own smallest step, halved
        above = (tops < t).sum()
        bound = bound + 2.002 * 2.0 ** -11 * np.abs(want) + 2.0 ** -32 * t * np.abs(hv).max() / above + 2.0 ** -25
        within(np.abs(got[s].reshape(1, 1, hd) - want), bound, (s, t))


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd,n_heads,window", [(64, 4, 1), (128, 2, 5), (256, 4, 32), (64, 8, 50), (512, 4, 31), (512, 2, 100)])
def test_small_windows(lib, combo, hd, n_heads, window):
    """windows of a few keys with rows enough in the call that it goes to the tiles; most of the rows are padding"""
    qk, ck = combo
    rng = np.random.default_rng(570 + window)
    n, hist, n_kv = [3, 96, 150, 1, 33, 0], [0, 40, 700, 600, 31, 9], 2
    lens = [a + b for a, b in zip(n, hist)]
    c = Cache(lib, rng, ck, hd, n_kv, 16, lens, extra=WIDE)
    k, v = rows(rng, sum(lens), n_kv, hd), rows(rng, sum(lens), n_kv, hd)
    c.store(k, v, lens, lens)
    m = rows_for_tiles(c, window, n_heads)
    assert m > sum(n) and tiles(c, window, m, n_heads)
    q, qf = cast(rows(rng, sum(n), n_heads, hd), qk)
    bits, got = run_chunk(lib, c, padded(q, m), qk, n, lens, window, n_heads, 0.1)
    assert (bits[sum(n):].view(np.uint8) == 0x3F).all()
    hk, hv = (pn.held(x, ck, hd).reshape(-1, n_kv, hd) for x in (k, v))
    at, key = pn.starts(n), pn.starts(lens)
    for s, (t, h) in enumerate(zip(n, hist)):
        for lo in range(0, t, 64):
            hi = min(t, lo + 64)
            first = [max(0, h + i + 1 - window) for i in range(lo, hi)]
            kk = slice(key[s] + first[0], key[s] + h + hi)
            qq = qf[at[s] + lo:at[s] + hi].reshape(hi - lo, n_heads, hd)
            want, bound = pn.attention(qq, hk[kk], hv[kk], np.array(first) - first[0], 0.1)
            bound = bound_of(bound, want, qq, hk[kk], hv[kk], qk, ck, 0.1)
            within(np.abs(got[at[s] + lo:at[s] + hi].reshape(hi - lo, n_heads, hd) - want), bound, (s, lo))


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd,window", [(64, 50), (128, 300), (256, 50), (512, 300), (512, 20)])
def test_pages_before_a_window(lib, combo, hd, window):
    """pages that no row sees any more: entries that are no page, that lie outside the pool, or another sequence's with
    infinities and NaN in them"""
    qk, ck = combo
    rng = np.random.default_rng(580 + window)
    page, t, new, n_heads = 16, 420, 20, 2
    c = Cache(lib, rng, ck, hd, 1, page, [t, t], extra=WIDE)
    k, v = rows(rng, 2 * t, 1, hd), rows(rng, 2 * t, 1, hd)
    c.store(k, v, [t, t], [t, t])
    q = cast(rows(rng, 2 * new, n_heads, hd), qk)[0]
    m = max(2 * new, rows_for_tiles(c, window, n_heads))
    assert tiles(c, window, m, n_heads)
    q = padded(q, m)
    a, af = run_chunk(lib, c, q, qk, [new, new], [t, t], window, n_heads, 0.1)
    assert np.isfinite(af[:2 * new]).all()
    gone = (t - new + 1 - window) // page
    good = c.table.copy()
    spare = np.setdiff1d(np.arange(c.pages), good)       # a page of no sequence: NaN, as Cache fills its pools
    for entry in (-1, c.pages, (1 << 31) - 1, -(1 << 31), int(spare[0])):
        c.table = good.copy()
        c.table[0, :gone] = entry
        c.dtable.write(c.table)
        b, _ = run_chunk(lib, c, q, qk, [new, new], [t, t], window, n_heads, 0.1)
        assert same_bits(a, b), entry
    c.table = good
    c.dtable.write(good)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd,window", [(64, 30), (256, 260), (256, 30), (512, 30), (512, 130)])
def test_bad_pages_and_windows(lib, combo, hd, window):
    """a page outside the pool under a window: NaN in the rows that see it, no bit of the others"""
    qk, ck = combo
    rng = np.random.default_rng(590 + window)
    n, hist, n_heads = [40, 200, 3], [50, 150, 300], 2
    lens = [a + b for a, b in zip(n, hist)]
    c = Cache(lib, rng, ck, hd, 1, 16, lens, extra=WIDE)
    x = rows(rng, sum(lens), 1, hd)
    c.store(x, x, lens, lens)
    m = max(sum(n), rows_for_tiles(c, window, n_heads))
    assert tiles(c, window, m, n_heads)
    q = padded(cast(rows(rng, sum(n), n_heads, hd), qk)[0], m)
    a, _ = run_chunk(lib, c, q, qk, n, lens, window, n_heads, 0.1)
    old = c.table.copy()
    c.table[1, 11], c.table[2, 0], c.table[2, 18] = c.pages, -5, c.pages + 7    # positions 176 .. 191; 0 .. 15, 288 .. 303
    c.dtable.write(c.table)
    b, bf = run_chunk(lib, c, q, qk, n, lens, window, n_heads, 0.1)
    c.table = old
    c.dtable.write(old)
    at = pn.starts(n)
    assert same_bits(a[:at[1]], b[:at[1]]) and same_bits(a[at[3]:], b[at[3]:])
    for s, bad in ((1, [(176, 191)]), (2, [(0, 15), (288, 303)])):
        p = np.arange(hist[s], lens[s])
        sees = np.zeros(len(p), bool)
        for lo, hi in bad:
            sees |= (p >= lo) & (p - window + 1 <= hi)
        one = slice(at[s], at[s + 1])
        assert np.isnan(bf[one][sees]).all() and same_bits(a[one][~sees], b[one][~sees])


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd", [64, 512])
def test_misfits(lib, combo, hd):
    """more rows than positions, past the table, past the rows, starts that do not ascend or lie anywhere: those rows stay
    as they are, the others are done; up to 64 sequences and more"""
    qk, ck = combo
    rng = np.random.default_rng(600 + hd)
    width = WIDE
    for seqs in (4, 100):
        c = Cache(lib, rng, ck, hd, 1, 16, [40] * seqs, extra=width)
        x = rows(rng, 40 * seqs, 1, hd)
        c.store(x, x, [40] * seqs, [40] * seqs)
        n = [6] * seqs
        q, qf = cast(rows(rng, 6 * seqs, 2, hd), qk)
        assert tiles(c, 0, len(q), 2)
        lens = [40, 5, c.table.shape[1] * 16 + 1, 40] + [40] * (seqs - 4)
        lens[-1] = 40 if seqs == 4 else -7
        bits, got = run_chunk(lib, c, q, qk, n, lens, 0, 2, 0.1)
        hx = pn.held(x, ck, hd).reshape(-1, 1, hd)
        for s in range(seqs):
            one = slice(6 * s, 6 * s + 6)
            if lens[s] != 40:
                assert (bits[one].view(np.uint8) == 0x3F).all()
                continue
            f, qq = hx[40 * s:40 * s + 40], qf[one].reshape(6, 2, hd)
            want, bound = pn.attention(qq, f, f, [0] * 6, 0.1)
            within(np.abs(got[one].reshape(6, 2, hd) - want), bound_of(bound, want, qq, f, f, qk, ck, 0.1), s)
        if seqs > 4:
            continue
        out = filled(lib, q.nbytes, 0x3F)
        dq, dl = dbuf(lib, q), dbuf(lib, np.array([40] * 4, np.int32))
        part = filled(lib, lib.L.g4_attn_chunk_paged_part_bytes(24, 2, 1, hd))
        for cu in ([0, 6, 5, -3, 200], [0, 6, 12, 30, 24], [-7, -1, 3, 2, 1 << 30], [0, 6, 6, 6, 24]):
            dcu = dbuf(lib, np.array(cu, np.int32))
            lib.g4_memset(out.ptr, 0x3F, out.nbytes)
            lib.g4_attn_chunk_paged(dq.ptr, 2 * hd, qk, *c.args(), dcu.ptr, dl.ptr, 4, 24, 0, 2, F(0.1), part.ptr, out.ptr, 2 * hd)
            lib.g4_sync()
            o = out.to_array(NPT[qk]).reshape(24, -1)
            may = np.zeros(24, bool)
            for s in range(4):
                if 0 <= cu[s] < cu[s + 1] <= 24:
                    may[cu[s]:cu[s + 1]] = True
            assert (o[~may].view(np.uint8) == 0x3F).all() and np.isfinite(back(o[may], qk)).all()


@pytest.mark.parametrize("combo", COMBOS, ids=str)
@pytest.mark.parametrize("hd", [64, 256, 512])
def test_common_prefix(lib, combo, hd):
    """sequences with the same first pages and rows of their own, cut into tiles: each what it would be alone"""
    qk, ck = combo
    rng = np.random.default_rng(610 + hd)
    page, n_heads = 16, 2
    table = np.full((2, 5 + WIDE), -1, np.int32)
    table[:, :5] = [[0, 1, 2, 3, 4], [0, 1, 2, 5, 6]]
    c = Cache(lib, rng, ck, hd, 1, page, None, table=table, pages=7)
    x = rows(rng, 48 + 20 + 27, 1, hd)
    c.store(x[:48], x[:48], [48, 0], [48, 48])
    c.store(x[48:], x[48:], [20, 27], [68, 75])
    q, qf = cast(rows(rng, 47, n_heads, hd), qk)
    assert tiles(c, 0, 47, n_heads)
    _, got = run_chunk(lib, c, q, qk, [20, 27], [68, 75], 0, n_heads, 0.1)
    for r0, r1 in ((0, 20), (20, 47)):
        f = pn.held(np.concatenate([x[:48], x[48 + r0:48 + r1]]), ck, hd).reshape(-1, 1, hd)
        qq = qf[r0:r1].reshape(-1, n_heads, hd)
        want, bound = pn.attention(qq, f, f, [0] * (r1 - r0), 0.1)
        within(np.abs(got[r0:r1].reshape(-1, n_heads, hd) - want), bound_of(bound, want, qq, f, f, qk, ck, 0.1), r0)


@pytest.mark.parametrize("combo", COMBOS, ids=str)
def test_ended_sequences(lib, combo):
    """many sequences without rows, at the front, at the end and between the others, whatever their lengths are"""
    qk, ck = combo
    rng = np.random.default_rng(620)
    hd, n_heads = 128, 2
    for seqs in (60, 900):
        n, lens = [0] * seqs, [int(x) for x in rng.choice([0, 0, 50, 70, -1, 1 << 30], seqs)]
        used = [seqs // 4, seqs // 2, seqs - 3]
        for s, (a, b) in zip(used, ((30, 60), (1, 64), (2, 2))):
            n[s], lens[s] = a, b
        c = Cache(lib, rng, ck, hd, 1, 16, [lens[s] if s in used else 0 for s in range(seqs)], extra=WIDE)
        k, v = rows(rng, 126, 1, hd), rows(rng, 126, 1, hd)
        ns = [lens[s] if s in used else 0 for s in range(seqs)]
        c.store(k, v, ns, ns)
        q, qf = cast(rows(rng, 33, n_heads, hd), qk)
        assert tiles(c, 0, 33, n_heads)
        _, got = run_chunk(lib, c, q, qk, n, lens, 0, n_heads, 0.1)
        hk, hv = (pn.held(x, ck, hd).reshape(-1, 1, hd) for x in (k, v))
        for (r0, r1), (k0, k1) in zip(((0, 30), (30, 31), (31, 33)), ((0, 60), (60, 124), (124, 126))):
            qq = qf[r0:r1].reshape(-1, n_heads, hd)
            want, bound = pn.attention(qq, hk[k0:k1], hv[k0:k1], [0] * (r1 - r0), 0.1)
            bound = bound_of(bound, want, qq, hk[k0:k1], hv[k0:k1], qk, ck, 0.1)
            within(np.abs(got[r0:r1].reshape(-1, n_heads, hd) - want), bound, (seqs, r0))
