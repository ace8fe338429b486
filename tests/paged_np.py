"""Plain forms of the paged cache and of the attentions over many sequences, in
64 bits (numpy), and the bounds their fp32 kernels are held to."""
import numpy as np

F32, F16, BF16, Q8 = 0, 1, 30, 1024
TYPES = (F32, F16, BF16, Q8)
# largest relative error of one rounding to the type
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def bf16_bits(x):
    """nearest-even bf16 bit patterns of float32 (infinities and NaN kept)"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    nan = (u & 0x7FFFFFFF) > 0x7F800000
    return np.where(nan, (u >> 16) | 0x40, r).astype(np.uint16)


def bf16_back(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def held(x, kind, hd):
    """what a cache of the type reads back for rows x [rows, heads * hd]"""
    x = np.ascontiguousarray(x, np.float32)
    if kind == F32:
        return x
    if kind == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    if kind == BF16:
        return bf16_back(bf16_bits(x))
    r = x.reshape(x.shape[0], -1, hd)
    with np.errstate(all="ignore"):
        d = (np.abs(r).max(-1, keepdims=True) / np.float32(127)).astype(np.float32)
        codes = np.where(d > 0, np.clip(np.rint(r / d), -127, 127), np.float32(0))
        d = np.where(np.isfinite(r).all(-1, keepdims=True), d, np.float32(np.nan))
        return (np.where(np.isnan(d), np.float32(0), codes) * d).astype(np.float32).reshape(x.shape)


def attention(q, k, v, first, scale):
    """(o, bound): q [rows, heads, hd] over keys first[i] .. last[i] (the last row sees the last key), k, v [keys, kv, hd];
    bound: what fp32 arithmetic may be off, see below"""
    rows, heads, hd = q.shape
    keys, kv = k.shape[:2]
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    at = np.arange(keys)
    last = np.arange(keys - rows, keys)
    seen = (at >= np.asarray(first)[:, None]) & (at <= last[:, None])
    for h in range(heads):
        g = h // (heads // kv)
        # keys outside are left out before any arithmetic on them
        for i in range(rows):
            ks, vs = k[seen[i], g], v[seen[i], g]
            s = scale * (ks @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vs
            # A score is a sum of hd products in at most hd / 8 + 16 steps of fp32, each off by 2^-24 of the sum of
            # magnitudes, and is scaled, shifted and exponentiated (four roundings of its size and the maximum's);
            # a weight's relative error is that of its score, once in the numerator and once in the denominator;
            # the weights' sums take at most keys + 64 further steps (merges among them).
            mags = abs(scale) * (np.abs(ks) @ np.abs(q[i, h])).max()
            rel = 2 * ((hd / 8 + 16) * mags + 4 * np.abs(s).max()) + len(ks) + 64
            bound[i, h] = rel * 2.0 ** -24 * (p @ np.abs(vs)) + 1e-37
    return out, bound


def starts(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def page_table(rng, lens, page, spare=2, extra=2):
    """(table, pages): pages of each sequence in no order, -1 past its last"""
    need = [-(-int(t) // page) for t in lens]
    perm = rng.permutation(sum(need) + spare).astype(np.int32)
    table = np.full((len(need), max(max(need), 1) + extra), -1, np.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = perm[at:at + c]
        at += c
    return table, sum(need) + spare
