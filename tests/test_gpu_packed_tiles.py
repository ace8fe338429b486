"""GPU parity of the attention of packed prompts where its tiles run: batches
of so many rows, keys and heads that the kernel for few rows does not take
them.  The attention block is main.c:1909-1950 of the reference."""
import numpy as np
import pytest

import paged_np as pn
import test_gpu_paged as base
from test_gpu_paged import NAN, cast, rows, run_prompt, within

pytestmark = pytest.mark.gpu

FEW = 1 << 18     # rows x keys x heads up to which the kernel for few rows is taken
KINDS = [(pn.F32, 64), (pn.F32, 128), (pn.F32, 256), (pn.F32, 512), (pn.F16, 128), (pn.F16, 512), (pn.BF16, 64),
         (pn.BF16, 256), (pn.BF16, 512)]


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


def in_tiles(m, window, heads):
    assert m * (min(m, window) if window else m) * heads > FEW


def check(lib, seed, kind, hd, n_heads, n_kv, n, window=0, pad=0, **kw):
    in_tiles(sum(n) + pad, window, n_heads)
    base.check_prompt(lib, seed, kind, hd, n_heads, n_kv, n, window=window, pad=pad, **kw)


@pytest.mark.parametrize("kind,hd", KINDS)
def test_strides(lib, kind, hd):
    """rows wider than their heads, rows past the last sequence"""
    check(lib, 500, kind, hd, 8, 2, [150, 1, 0, 70], extra=8, pad=5)


@pytest.mark.parametrize("kind,hd", KINDS)
@pytest.mark.parametrize("window", [33, 100])
def test_windows(lib, kind, hd, window):
    """windows shorter than the sequences, which end inside tiles"""
    check(lib, 501, kind, hd, 8, 2, [700, 300, 40, 1], window=window, some=3)


@pytest.mark.parametrize("kind,hd", [(pn.F32, 64), (pn.F32, 512), (pn.BF16, 256), (pn.F16, 512)])
def test_window_of_one(lib, kind, hd):
    """every row sees itself only"""
    check(lib, 502, kind, hd, 48, 16 if hd < 512 else 2, [5000, 480, 1, 31], window=1, some=32)


@pytest.mark.parametrize("kind,hd", KINDS)
def test_extremes(lib, kind, hd):
    """weights on one key, equal weights, a negative scale, a scale of zero, magnitudes far from 1"""
    n = [230, 20]
    check(lib, 503, kind, hd, 8, 2, n, gain=60.0, scale=1.0)
    check(lib, 504, kind, hd, 8, 2, n, gain=0.0, scale=1.0)
    check(lib, 505, kind, hd, 8, 2, n, scale=-0.09)
    check(lib, 506, kind, hd, 8, 2, n, scale=0.0)
    if kind != pn.F16:
        check(lib, 507, kind, hd, 8, 2, n, gain=1e-18, scale=1e17)


@pytest.mark.parametrize("n_heads,n_kv", [(1, 1), (3, 3), (5, 1), (10, 2), (12, 1), (20, 1), (24, 8)])
def test_heads(lib, n_heads, n_kv):
    """one head to twenty on a kv head"""
    for kind, hd in ((pn.F32, 128), (pn.F32, 512), (pn.BF16, 64), (pn.BF16, 512)):
        check(lib, 510 + n_heads, kind, hd, n_heads, n_kv, [400, 1, 165, 100], some=2)


@pytest.mark.parametrize("kind,hd", [(pn.F32, 64), (pn.F32, 256), (pn.F32, 512), (pn.F16, 512), (pn.BF16, 256)])
def test_many(lib, kind, hd):
    """more than 64 sequences, empty ones among them"""
    rng = np.random.default_rng(520)
    n = [int(x) for x in rng.integers(0, 30, 90)] + [170]
    check(lib, 520, kind, hd, 4, 2, n, window=0)
    check(lib, 521, kind, hd, 12, 2, n, window=20)


def test_lengths(lib):
    """sequences of 1 to 136 rows one after the other, a window that ends inside tiles"""
    for kind, hd in ((pn.F32, 64), (pn.F32, 512), (pn.BF16, 64), (pn.BF16, 512)):
        check(lib, 522, kind, hd, 12, 2, list(range(1, 141, 9)), window=33)


def rounded(kind, want, bound, v):
    """16 bits: the bound with weights and results rounded to the type, as the types' test derives it"""
    if kind == pn.F32:
        return bound
    big = np.abs(v).max()
    return bound + pn.HALF[kind] * (np.abs(want) + 1.01 * big) + 2.0 ** -25 * len(v) * big


@pytest.mark.parametrize("kind,hd", KINDS)
@pytest.mark.parametrize("window", [0, 60])
def test_not_finite(lib, kind, hd, window):
    """infinities and NaN in rows of other sequences, in rows past the last sequence, in later rows of the same sequence
    and before the window do not matter to a row that does not see them; a row that sees them has NaN or infinities in
    the heads that do"""
    rng = np.random.default_rng(530)
    n_heads, n_kv, n = 16, 2, [150, 145, 60]
    m, cu = sum(n) + 6, pn.starts(n)
    in_tiles(m, window, n_heads)
    q, k, v = (cast(rows(rng, m, h, hd), kind)[1] for h in (n_heads, n_kv, n_kv))
    want, bound = [np.empty((m, n_heads, hd)) for _ in range(2)]
    for s, t in enumerate(n):
        r = slice(cu[s], cu[s + 1])
        w, b = pn.attention(q[r].reshape(t, n_heads, hd), k[r].reshape(t, n_kv, hd), v[r].reshape(t, n_kv, hd),
                            [max(0, i + 1 - window) if window else 0 for i in range(t)], 0.1)
        want[r], bound[r] = w, rounded(kind, w, b, v[r])
    q2, k2, v2 = q.copy(), k.copy(), v.copy()
    k2[cu[3]:] = v2[cu[3]:] = q2[cu[3]:] = NAN
    v2[150 + 37, hd + 3] = np.inf         # row 37 of sequence 1, kv head 1
    k2[150 + 40, 5] = NAN                 # row 40, kv head 0
    k2[2, hd + 1] = -np.inf               # row 2 of sequence 0, kv head 1
    q2[cu[2] + 20, hd * 3 + 1] = NAN      # row 20 of sequence 2, q head 3
    got = run_prompt(lib, *(cast(x, kind)[0] for x in (q2, k2, v2)), kind, cu, m, window, n_heads, n_kv, hd, 0.1)[1]
    got = got.reshape(m, n_heads, hd)
    hit = np.zeros((m, n_heads), bool)
    for row, heads, end in ((187, slice(8, 16), 295), (190, slice(0, 8), 295), (2, slice(8, 16), 150)):
        hit[row:min(end, row + window) if window else end, heads] = True
    hit[cu[2] + 20, 3] = True
    # K and q: NaN; V: the element is not finite, the others may be NaN
    assert np.isnan(got[190:min(295, 190 + window) if window else 295, :8]).all() and np.isnan(got[cu[2] + 20, 3]).all()
    assert not np.isfinite(got[187:min(295, 187 + window) if window else 295, 8:, 3]).any()
    keep = ~hit[:cu[3]]
    within(np.abs(got[:cu[3]] - want[:cu[3]])[keep], bound[:cu[3]][keep], (kind, hd))
    assert np.isfinite(got[cu[3]:]).all()      # left as they were


@pytest.mark.parametrize("kind,hd", [(pn.F32, 64), (pn.F32, 512), (pn.BF16, 64), (pn.BF16, 512)])
def test_starts_that_do_not_fit(lib, kind, hd):
    """row starts that are not ascending or run past m: those sequences' rows are left as they are, the others' not"""
    rng = np.random.default_rng(540)
    m, n_heads, n_kv = 420, 4, 2
    in_tiles(m, 0, n_heads)
    q, k, v = (cast(rows(rng, m, h, hd), kind) for h in (n_heads, n_kv, n_kv))
    many = [2 * i for i in range(70)]
    for cu, good in (([0, 200, 900, 290, -5], [(0, 200)]), ([3, 40, 300, 421], [(3, 40), (40, 300)]),
                     (many + [360, 500, 600], [(2 * i, 2 * i + 2) for i in range(69)] + [(138, 360)])):
        bits, got = run_prompt(lib, q[0], k[0], v[0], kind, cu, m, 0, n_heads, n_kv, hd, 0.1)
        left = np.ones(m, bool)
        for a, b in good:
            left[a:b] = False
            t = b - a
            want, bound = pn.attention(q[1][a:b].reshape(t, n_heads, hd), k[1][a:b].reshape(t, n_kv, hd),
                                       v[1][a:b].reshape(t, n_kv, hd), [0] * t, 0.1)
            bound = rounded(kind, want, bound, v[1][a:b])
            within(np.abs(got[a:b].reshape(t, n_heads, hd) - want), bound, (a, b))
        untouched = np.full(1, 0x3F3F3F3F, np.uint32).view(bits.dtype)[0]
        assert (bits[left] == untouched).all()


@pytest.mark.parametrize("kind,hd", [(pn.F32, 64), (pn.BF16, 512)])
def test_starts_that_do_not_fit_few_rows(lib, kind, hd):
    """the same in the kernel for few rows"""
    rng = np.random.default_rng(541)
    m, n_heads, n_kv = 40, 4, 2
    q, k, v = (cast(rows(rng, m, h, hd), kind) for h in (n_heads, n_kv, n_kv))
    for cu, a, b in (([0, 10, 300, 290, -5], 0, 10), ([2, 30, 41], 2, 30)):
        bits, got = run_prompt(lib, q[0], k[0], v[0], kind, cu, m, 0, n_heads, n_kv, hd, 0.1)
        t = b - a
        want, bound = pn.attention(q[1][a:b].reshape(t, n_heads, hd), k[1][a:b].reshape(t, n_kv, hd),
                                   v[1][a:b].reshape(t, n_kv, hd), [0] * t, 0.1)
        within(np.abs(got[a:b].reshape(t, n_heads, hd) - want), rounded(kind, want, bound, v[1][a:b]), (a, b))
        left = np.r_[0:a, b:m]
        assert (bits[left] == np.full(1, 0x3F3F3F3F, np.uint32).view(bits.dtype)[0]).all()


def test_serving(lib):
    """prompts of a ragged batch (attention, cache written), then steps of one token each: every output equals a plain
    forward over the whole sequences"""
    rng = np.random.default_rng(550)
    hd, n_heads, n_kv, page, window, scale = 256, 8, 2, 16, 100, 1 / 16
    n, steps = [150, 1, 130, 64], 5
    in_tiles(sum(n), window, n_heads)
    lens = np.array(n)
    total = [t + steps for t in n]
    seqs = [tuple(rows(rng, t, h, hd) for h in (n_heads, n_kv, n_kv)) for t in total]
    for kind in (pn.F32, pn.Q8):
        c = base.Cache(lib, rng, kind, hd, n_kv, page, total)
        q, k, v = (np.concatenate([s[i][:t] for s, t in zip(seqs, n)]) for i in range(3))
        o = run_prompt(lib, q, k, v, pn.F32, pn.starts(n), len(q), window, n_heads, n_kv, hd, scale)[1]
        got = [[x] for x in np.split(o, pn.starts(n)[1:-1])]
        c.store(k, v, n, n)
        for i in range(steps):
            q, k, v = (np.stack([s[j][t + i] for s, t in zip(seqs, n)]) for j in range(3))
            c.store(k, v, [1] * 4, lens + i + 1)
            o = base.run_decode(lib, c, q, lens + i + 1, n_heads, window, scale)
            for s in range(4):
                got[s].append(o[s:s + 1])
        for s, t in enumerate(n):
            qs, ks, vs = seqs[s]
            o = np.concatenate(got[s]).reshape(total[s], n_heads, hd)
            hk, hv = pn.held(ks, kind, hd), pn.held(vs, kind, hd)
            first = [max(0, i + 1 - window) for i in range(total[s])]
            for lo, hi, kk, vv in ((0, t, ks, vs), (t, total[s], hk, hv)):
                want, bound = pn.attention(qs[lo:hi].reshape(hi - lo, n_heads, hd), kk[:hi].reshape(hi, n_kv, hd),
                                           vv[:hi].reshape(hi, n_kv, hd), first[lo:hi], scale)
                within(np.abs(o[lo:hi] - want), bound, (s, lo))


def fp32_bound(q, k, v, want_bound, first, scale):
    """(want, bound) of one sequence's fp32 rows whose sizes differ much from key to key: pn.attention's with what the
    tiles may be off beside it, see below"""
    want, bound = want_bound
    t, n_heads, _ = q.shape
    big = np.abs(v).max(-1).repeat(n_heads // v.shape[1], 1).astype(np.float64)
    for i in range(t):
        seen = slice(first[i], i + 1)
        for h in range(n_heads):
            sc = scale * (k[seen, h // (n_heads // k.shape[1])].astype(np.float64) @ q[i, h])
            p = np.exp(sc - sc.max())
            pb = p * big[seen, h]
            # An element of V is met within 2^-39 of its row's largest; a weight times its V row's power of two is held
            # as two fp16, the largest of them at 2^11 or more and each within 2^-25: times V's scaled elements, below
            # 2^15, that is 2^-10 a key where the largest stands for 2^11 * 2^14 at least, 2^-35 of it.
            bound[i, h] += (2.0 ** -38 * pb.sum() + 2.0 ** -35 * len(p) * pb.max()) / p.sum()
            # Rows of V below 2^-76 have the scale of 2^-76, 2^90: halves within 2^-25 of the scaled row are 2^-115 of V.
            bound[i, h] += 2.0 ** -115
            # A score has the row's exponent (-90 to 113) added and the maximum taken off: two roundings of numbers
            # below 256, 2^-17 each and times ln 2 in a weight, met in the numerator and in the denominator.
            bound[i, h] += 4 * np.log(2) * 2.0 ** -17 * (p @ np.abs(v[seen, h // (n_heads // v.shape[1])])) / p.sum()
    return want, bound


def check_far(lib, hd, k, v, gain, window=0, seed=560):
    rng = np.random.default_rng(seed)
    t, n_heads, n_kv = len(v), 16, 2
    in_tiles(t, window, n_heads)
    q = rows(rng, t, n_heads, hd) * np.float32(gain)
    _, got = run_prompt(lib, q, k, v, pn.F32, [0, t], t, window, n_heads, n_kv, hd, hd ** -0.5)
    first = [max(0, i + 1 - window) if window else 0 for i in range(t)]
    q, k, v = (x.reshape(t, -1, hd) for x in (q, k, v))
    want, bound = fp32_bound(q, k, v, pn.attention(q, k, v, first, hd ** -0.5), first, hd ** -0.5)
    within(np.abs(got.reshape(t, n_heads, hd) - want), bound, hd)


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("top", [61, 62, 100, 126])
@pytest.mark.parametrize("big_first", [False, True])
def test_values_far_apart(lib, hd, top, big_first):
    """V rows of zeros beside one of 2^62 and more, in front of it and behind it, with equal scores and with scores far
    apart: a row of zeros takes its share of the weights whatever the others hold"""
    rng = np.random.default_rng(561)
    t = 150
    k, v = rows(rng, t, 2, hd), np.zeros((t, 2 * hd), np.float32)
    at = 3 if big_first else 100
    v[at] = np.float32(1.5 * 2.0 ** top)
    check_far(lib, hd, k, v, 0.0)
    check_far(lib, hd, k, v, 6.0)
    # tiny rows, in tiles of their own and beside large ones, and a window
    v = rows(rng, t, 2, hd) * np.exp2(np.where(np.arange(t) // 40 % 2 == big_first, top - 3, -103)).astype(np.float32)[:, None]
    v[rng.integers(0, t, 9)] = 0
    check_far(lib, hd, k, v, 3.0)
    check_far(lib, hd, np.concatenate([k] * 3), np.concatenate([v] * 3), 3.0, window=70)


@pytest.mark.parametrize("hd,window", [(64, 40), (256, 40), (512, 40)])
def test_magnitudes(lib, hd, window):
    """fp32 rows whose sizes differ by 2^60 from key to key and by 2^20 within a row, under a window"""
    rng = np.random.default_rng(570 + hd)
    t = 430
    k, v = rows(rng, t, 2, hd), rows(rng, t, 2, hd)
    v *= np.exp2(rng.integers(-30, 31, (t, 2 * hd // 64))).repeat(64, 1).astype(np.float32)
    v *= np.exp2(rng.integers(-10, 11, v.shape)).astype(np.float32)
    k *= np.exp2(rng.integers(-6, 3, (t, 1))).astype(np.float32)
    k[rng.integers(0, t, 12)] *= np.float32(20)
    v[7] = v[200] = k[31] = 0
    check_far(lib, hd, k, v, 1.0, window=window)


@pytest.mark.parametrize("hd", [64, 256, 512])
def test_values_at_the_limit(lib, hd):
    """bf16 V so large that the keys together stay just below fp32's largest number, under scores that rise by 2^7.9 from
    one of a wave's tiles to the next"""
    t, n_heads, n_kv, top = 400, 8, 2, 119
    in_tiles(t, 0, n_heads)
    assert t * 2.0 ** top < float(np.finfo(np.float32).max) < t * 2.0 ** (top + 1)
    k = np.zeros((t, n_kv, hd), np.float32)
    for i in range(t):
        k[i, :, :i // 64] = 1
    v = np.full((t, n_kv * hd), 2.0 ** top, np.float32)
    v *= np.random.default_rng(580).choice(np.array([1, -1], np.float32), n_kv * hd)
    q = np.zeros((t, n_heads, hd), np.float32)
    q[:, :, :16] = 5.46875
    _, got = run_prompt(lib, *(cast(x.reshape(t, -1), pn.BF16)[0] for x in (q, k, v)), pn.BF16, [0, t], t, 0, n_heads, n_kv, hd,
                        1.0)
    want, bound = pn.attention(q, k, v.reshape(t, n_kv, hd), [0] * t, 1.0)
    within(np.abs(got.reshape(t, n_heads, hd) - want), rounded(pn.BF16, want, bound, v), hd)
