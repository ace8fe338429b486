"""GPU parity of the attention of packed prompts where its tiles run: batches
of so many rows, keys and heads that the kernel for few rows does not take
them.  The attention block is main.c:1909-1950 of the reference."""
import numpy as np
import pytest

import paged_np as pn
from test_gpu_paged import cast, rows, run_prompt, within

pytestmark = pytest.mark.gpu

FEW = 1 << 18     # rows x keys x heads up to which the kernel for few rows is taken


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


def in_tiles(m, window, heads):
    assert m * (min(m, window) if window else m) * heads > FEW


def rounded(kind, want, bound, v):
    """16 bits: the bound with weights and results rounded to the type, as the types' test derives it"""
    if kind == pn.F32:
        return bound
    big = np.abs(v).max()
    return bound + pn.HALF[kind] * (np.abs(want) + 1.01 * big) + 2.0 ** -25 * len(v) * big


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
