"""The measured cases of the operators that take a server's step from the
projections to the attention: norms of q, k and v heads with the rotation at
each row's own position (rows out), the same straight into the paged cache, and
the attention of chunks of new rows of every sequence over that cache.

Where `own` is false they are computed from elementary torch operations in 32
bits; where it is true they go through the C ABI (include/g4hip.h).
Head layouts, window and context are the E4B shape's (8 query / 2 KV heads of
256 with a window of 512, or of 512 without one); the drawn cases take others too.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SIZES = {"F32": 4, "F16": 2, "BF16": 2, "Q8": 1}
TORCH = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
EPS = 1e-6
# types of q rows that each type of cache is attended with
Q_TYPES = {"F32": ["F32"], "F16": ["F16", "F32"], "BF16": ["BF16", "F32"], "Q8": ["BF16", "F32"]}


def listed():
    return [
        # prompts of twelve conversations on a sliding-window layer, made ready for 16-bit attention; the batch is padded
        {"name": "post_prompts", "kind": "post", "q": "BF16", "kv_rows": True, "hd": 256, "rot": 256, "heads": 8, "kv": 2,
         "seqs": 12, "lo": 5, "hi": 2048, "hlo": 0, "hhi": 0, "pad": 13, "mix": 1},
        # one token each of 48 conversations on a global layer that shares another one's K and V: q alone
        {"name": "post_tokens", "kind": "post", "q": "F32", "kv_rows": False, "hd": 512, "rot": 512, "heads": 8, "kv": 2,
         "seqs": 48, "lo": 1, "hi": 1, "hlo": 16, "hhi": 30000, "pad": 0, "mix": 2},
        # one token each of 48 conversations on a sliding-window layer: latency
        {"name": "append_tokens", "kind": "append", "type": "F16", "q": "F32", "hd": 256, "rot": 256, "heads": 8, "kv": 2,
         "page": 16, "seqs": 48, "lo": 1, "hi": 1, "hlo": 16, "hhi": 3000, "pad": 0, "mix": 3},
        # chunks of nine prompts, first and later ones, on a global layer
        {"name": "append_chunks", "kind": "append", "type": "BF16", "q": "BF16", "hd": 512, "rot": 512, "heads": 8, "kv": 2,
         "page": 64, "seqs": 9, "lo": 7, "hi": 1024, "hlo": 0, "hhi": 3000, "pad": 5, "mix": 4},
        # a long prompt in the engine's 32 bits
        {"name": "append_long", "kind": "append", "type": "F32", "q": "F32", "hd": 256, "rot": 256, "heads": 8, "kv": 2,
         "page": 32, "seqs": 1, "lo": 8191, "hi": 8191, "hlo": 0, "hhi": 0, "pad": 0, "mix": 5},
        # the next message of one chat on a sliding-window layer: latency
        {"name": "chunk_turn", "kind": "chunk", "type": "BF16", "q": "BF16", "hd": 256, "heads": 8, "kv": 2, "page": 16,
         "seqs": 1, "lo": 23, "hi": 23, "hlo": 1200, "hhi": 1200, "big": 0, "pad": 0, "window": 512, "mix": 6},
        # drafts of a few tokens of 32 conversations, checked in one step over a cache in codes
        {"name": "chunk_drafts", "kind": "chunk", "type": "Q8", "q": "F32", "hd": 512, "heads": 8, "kv": 2, "page": 64,
         "seqs": 32, "lo": 4, "hi": 8, "hlo": 100, "hhi": 6000, "big": 0, "pad": 0, "window": 0, "mix": 7},
        # a server's mixed step on a global layer: a chunk of one prompt beside one token each of forty conversations
        {"name": "chunk_mixed", "kind": "chunk", "type": "BF16", "q": "BF16", "hd": 512, "heads": 8, "kv": 2, "page": 64,
         "seqs": 40, "lo": 1, "hi": 1, "hlo": 100, "hhi": 8000, "big": 471, "pad": 3, "window": 0, "mix": 8},
        # chunks of nine prompts on a sliding-window layer, in the engine's 32 bits
        {"name": "chunk_window", "kind": "chunk", "type": "F32", "q": "F32", "hd": 256, "heads": 8, "kv": 2, "page": 32,
         "seqs": 9, "lo": 60, "hi": 1500, "hlo": 1, "hhi": 9000, "big": 0, "pad": 11, "window": 512, "mix": 9},
        # two documents that go on, fp32 rows over a cache in 16 bits, without a window
        {"name": "chunk_pair", "kind": "chunk", "type": "F16", "q": "F32", "hd": 256, "heads": 8, "kv": 2, "page": 32,
         "seqs": 2, "lo": 600, "hi": 900, "hlo": 3000, "hhi": 9000, "big": 0, "pad": 0, "window": 0, "mix": 10},
        # a question of 250 tokens about a document, global layer in the engine's 32 bits
        {"name": "chunk_document", "kind": "chunk", "type": "F32", "q": "F32", "hd": 512, "heads": 8, "kv": 2, "page": 64,
         "seqs": 1, "lo": 250, "hi": 250, "hlo": 16001, "hhi": 16001, "big": 0, "pad": 0, "window": 0, "mix": 11},
        # the last chunk of a prompt of 33000 tokens on a global layer
        {"name": "chunk_last", "kind": "chunk", "type": "BF16", "q": "BF16", "hd": 512, "heads": 8, "kv": 2, "page": 64,
         "seqs": 1, "lo": 512, "hi": 512, "hlo": 32488, "hhi": 32488, "big": 0, "pad": 0, "window": 0, "mix": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) if lo < hi else lo


def draw(rng):
    kind = rng.choice(["post", "append", "append", "chunk", "chunk", "chunk", "chunk"])
    heads, kv = rng.choice([(8, 2), (8, 2), (4, 4), (8, 1), (16, 4), (24, 8), (10, 2), (12, 1), (20, 1), (3, 3)])
    hd = rng.choice([64, 128, 256, 256, 512, 512])
    case = {"kind": kind, "hd": hd, "heads": heads, "kv": kv, "seqs": _log(rng, 1, 48), "pad": rng.choice([0, 0, 1, 37]),
            "mix": rng.randint(0, 10 ** 6)}
    # rows of all sequences together, and tokens in the pools: as many numbers as the listed cases have
    most = min(3000 if kind == "chunk" else 8191, 25000000 // ((heads + 2 * kv) * hd))
    hi = max(1, most // case["seqs"])
    case["hi"] = hi = _log(rng, max(1, hi // 256), hi)
    case["lo"] = _log(rng, 1, hi)
    pool = 32000000 // (kv * hd) - case["seqs"] * hi
    case["hhi"] = min(pool // (case["seqs"] + 1), rng.choice([0, 1, _log(rng, 2, 4000), _log(rng, 100, 32000)]))
    if kind == "post":
        case.update(q=rng.choice(["F32", "F16", "BF16"]), kv_rows=rng.choice([True, True, False]))
    else:
        case["page"] = rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        # codes are rounded far more coarsely than 32 bits are off, so that one of a few hundred thousand lands elsewhere:
        # a chunk's attention has them
        case.update(type=rng.choice(["F32", "F16", "BF16"]), q=rng.choice(["F32", "F16", "BF16"]))
    if kind != "chunk":
        case["rot"] = rng.choice([hd, hd, hd // 2])
    else:
        case["type"] = rng.choice(["F32", "F16", "BF16", "Q8"])
        case["q"] = rng.choice(Q_TYPES[case["type"]])
        case["window"] = rng.choice([0, 0, 512, _log(rng, 1, 2000)])
        case["big"] = rng.choice([0, 0, _log(rng, 1, max(1, most - case["seqs"] * hi))])
        # pairs of rows and keys: as many as the largest listed case has
        rows = case["seqs"] * hi + case["big"]
        case["hhi"] = min(case["hhi"], 270000000000 // (4 * rows * heads * hd) - max(hi, case["big"]))
    case["hhi"] = max(0, case["hhi"])
    case["hlo"] = min(case["hhi"], rng.choice([0, 1, _log(rng, 2, 500)]))
    return case


# ---------------------------------------------------------------------------
# sizes and inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """(new rows, earlier tokens) of each sequence; big: one more sequence, of so many rows, among them"""
    rng = random.Random(case["mix"])
    n = [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    if case.get("big"):
        n.insert(rng.randint(0, len(n)), case["big"])
    had = [_log(rng, max(1, case["hlo"]), case["hhi"]) if case["hhi"] > case["hlo"] else case["hlo"] for _ in n]
    return n, had


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 31)


def _heads(g, rows, heads, hd, gain=1.0):
    """heads as their norms leave them, of unit rms, a few dims of every head larger; gain: a factor, or one a head"""
    x = torch.randn((rows, heads, hd), device="cuda", generator=g)
    x *= torch.rand((heads, hd), device="cuda", generator=g) * 1.5 + 0.25
    x = x / x.square().mean(-1, keepdim=True).sqrt()
    return (x * gain).reshape(rows, heads * hd)


def _raw(g, rows, heads, hd):
    """heads as the projections leave them: rows of other sizes, some dims larger"""
    x = torch.randn((rows, heads, hd), device="cuda", generator=g)
    x *= torch.rand((heads, hd), device="cuda", generator=g) * 1.5 + 0.25
    x *= torch.exp(torch.randn((rows, heads, 1), device="cuda", generator=g))
    return x.reshape(rows, heads * hd)


def _post_inputs(case, seed):
    """rows q, k, v as projections leave them, norm weights (K's carry hd^-1/2: the attention scale is 1), the (cos, sin)
    pairs of every position, as fp32 [positions, rot / 2, 2]"""
    n, had = _lengths(case)
    g = _gen(seed)
    rows, hd = sum(n) + case["pad"], case["hd"]
    q, k, v = (_raw(g, rows, h, hd) for h in (case["heads"], case["kv"], case["kv"]))
    qw = torch.rand(hd, device="cuda", generator=g) * 1.5 + 0.25
    kw = (torch.rand(hd, device="cuda", generator=g) * 1.5 + 0.25) * hd ** -0.5
    half = case["rot"] // 2
    turn = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    at = torch.arange(max(a + b for a, b in zip(n, had)), device="cuda", dtype=torch.float64)[:, None] * turn
    tab = torch.stack([torch.cos(at), torch.sin(at)], -1).float()
    return n, had, q, k, v, qw, kw, tab


def _chunk_inputs(case, seed):
    """q rows, from heads that look at everything to heads that look at a few keys, and K, V rows of all positions"""
    n, had = _lengths(case)
    g = _gen(seed)
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    q = _heads(g, sum(n) + case["pad"], heads, hd, torch.linspace(0.5, 5.0, heads, device="cuda")[:, None]).to(TORCH[case["q"]])
    rows = sum(n) + sum(had)
    return n, had, q, _heads(g, rows, kv, hd, hd ** -0.5), _heads(g, rows, kv, hd)


def _starts(n):
    cu = [0]
    for i in n:
        cu.append(cu[-1] + i)
    return cu


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(case, total, seed):
    """(table, pages in all): the pages that hold total[s] tokens of each sequence, in no order, as a pool that has been
    in use for some time gives them out; entries past a sequence's last page hold -1"""
    page = case["page"]
    need = [-(-t // page) for t in total]
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed * 31 + 5), dtype=torch.int32)
    table = torch.full((len(total), max(need) + 2), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = perm[at:at + c]
        at += c
    return table.cuda(), pages


# ---------------------------------------------------------------------------
# an append's outputs are the pools as they lie in memory: [pages, kv, blocks of 16 tokens, 16 hd elements] in the
# library's order (gemma4.c_amd/csrc/g4_kvpage.h)
# ---------------------------------------------------------------------------
def _place(slot, hd, size, is_v):
    """element of (token slot % 16, each dim) in its block: [tokens, hd]"""
    t, d = (slot % 16)[:, None], torch.arange(hd, device=slot.device)
    e = 16 // size
    if is_v:
        w = 64 // size
        return (d // w * 64 + t // 4 * 16 + d % 16) * e + d % w // 16 * 4 + t % 4
    return (d // (4 * e) * 64 + d // e % 4 * 16 + t) * e + d % e


def _put(pool, x, pages, slots, is_v):
    """rows x [tokens, kv, hd] into their pages"""
    kv, hd = x.shape[1:]
    at = _place(slots, hd, pool.element_size(), is_v)[:, None, :]
    pool[pages[:, None, None], torch.arange(kv, device=x.device)[:, None], (slots // 16)[:, None, None], at] = x.to(pool.dtype)


def _pools(case, pages):
    shape = (pages, case["kv"], case["page"] // 16, 16 * case["hd"])
    return [torch.zeros(shape, dtype=TORCH[case["type"]], device="cuda") for _ in range(2)]


# ---------------------------------------------------------------------------
# a chunk's plain form: a cache of [pages, page, kv, hd] values or codes, and a scale for each token and head of codes
# ---------------------------------------------------------------------------
def _plain_encode(x, case):
    x = x.reshape(x.shape[0], case["kv"], case["hd"])
    if case["type"] != "Q8":
        return x.to(TORCH[case["type"]]), None
    d = x.abs().amax(-1, keepdim=True)
    d = d / torch.full_like(d, 127.0)       # a division, which torch makes a product where the divisor is a number
    codes = torch.where(d == 0, torch.zeros_like(x), torch.round(x / d))
    return codes.to(torch.int8), d


def _plain_pool(case, pages):
    shape = (pages, case["page"], case["kv"], case["hd"])
    if case["type"] == "Q8":
        return (torch.zeros(shape, dtype=torch.int8, device="cuda"), torch.zeros(shape[:3] + (1,), device="cuda"))
    return (torch.zeros(shape, dtype=TORCH[case["type"]], device="cuda"), None)


def _plain_places(table, page, cu, lens, rows):
    """(page, slot, position) of packed rows: the last n of the lens[s] tokens of each sequence, one after the other"""
    cu = cu.long()
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), cu[1:] - cu[:-1], output_size=rows)
    p = torch.arange(rows, device="cuda") + (lens.long() - cu[1:])[seq]
    return (table[seq, p // page].long(), p % page, p) if table is not None else (None, None, p)


def _plain_attention(q, k, v, first, last):
    """q [rows, heads, hd] over the keys first[i]..last[i] of row i, k and v [keys, kv, hd], in 32 bits"""
    rows, heads, hd = q.shape
    keys, kv, _ = k.shape
    qg = q.float().reshape(rows, kv, heads // kv, hd).permute(1, 2, 0, 3).reshape(kv, heads // kv * rows, hd)
    s = torch.matmul(qg, k.float().permute(1, 2, 0).contiguous()).reshape(kv, heads // kv, rows, keys)
    at = torch.arange(keys, device=q.device)
    s = s.masked_fill((at < first[:, None]) | (at > last[:, None]), -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(kv, heads // kv * rows, keys)
    o = torch.matmul(p, v.float().permute(1, 0, 2).contiguous())
    return o.reshape(heads, rows, hd).permute(1, 0, 2)


def _plain_post(x, heads, hd, weight, cs):
    """norm of each head, with its weight and the rotation of its first pairs where there are any; [rows, heads, hd]"""
    x = x.reshape(len(x), heads, hd)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    if weight is None:
        return x
    x = x * weight
    half = cs.shape[1]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., :half], x[..., hd // 2:hd // 2 + half]
    y = x.clone()
    y[..., :half] = a * c - b * s
    y[..., hd // 2:hd // 2 + half] = a * s + b * c
    return y


# ---------------------------------------------------------------------------
def prepare(case, seed):
    kind = case["kind"]
    st = {"kind": kind, "case": case}
    if own:
        if os.path.join(ROOT, "gemma4.c_amd") not in sys.path:
            sys.path.insert(0, os.path.join(ROOT, "gemma4.c_amd"))
        import g4
        st["lib"] = lib = g4.Lib.get()
        lib.init(0)
        st["t"] = {"F32": g4.F32, "F16": g4.F16, "BF16": g4.BF16, "Q8": g4.KV_Q8}
    if kind == "chunk":
        n, had, st["q"], k, v = _chunk_inputs(case, seed)
        st["out"] = torch.zeros_like(st["q"])
    else:
        n, had, *x = _post_inputs(case, seed)
        st.update(zip(("q", "k", "v", "qw", "kw", "tab"), x))
        outs = ["q"] + (["k", "v"] if kind == "post" and case["kv_rows"] else [])
        st["out"] = {a: torch.zeros(st[a].shape, dtype=TORCH[case["q"]], device="cuda") for a in outs}
    total = [a + b for a, b in zip(n, had)]
    st.update(n=n, cu=_ints(_starts(n)), lens=_ints(total))
    if kind == "append":
        st["table"], st["pages"] = _table(case, total, seed)
        st["out"]["kp"], st["out"]["vp"] = _pools(case, st["pages"])
    elif kind == "chunk":
        st["table"], st["pages"] = _table(case, total, seed)
        every = _ints(_starts(total))
        if own:
            size = lib.L.g4_kv_pool_bytes(st["t"][case["type"]], st["pages"], case["page"], case["kv"], case["hd"])
            st["pools"] = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
            size = lib.L.g4_attn_chunk_paged_part_bytes(st["q"].shape[0], case["heads"], case["kv"], case["hd"])
            st["part"] = torch.empty(size, dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            lib.g4_kv_page_store(*_own_pool(st), k.data_ptr(), v.data_ptr(), k.shape[1], every.data_ptr(),
                                 st["lens"].data_ptr(), len(n), k.shape[0])
            lib.g4_sync()
        else:
            st["pools"] = [_plain_pool(case, st["pages"]) for _ in range(2)]
            pages, slots, _ = _plain_places(st["table"], case["page"], every, st["lens"], len(k))
            for pool, x in zip(st["pools"], (k, v)):
                codes, d = _plain_encode(x, case)
                pool[0][pages, slots] = codes
                if d is not None:
                    pool[1][pages, slots] = d
    torch.cuda.synchronize()
    return st


def _own_pool(st):
    """the arguments that name a pool and the pages of its sequences"""
    c = st["case"]
    kp, vp = st["pools"] if st["kind"] == "chunk" else (st["out"]["kp"], st["out"]["vp"])
    return (kp.data_ptr(), vp.data_ptr(), st["t"][c["type"]], st["pages"], c["page"], c["kv"], c["hd"],
            st["table"].data_ptr(), st["table"].shape[1])


def run(st):
    kind, case, out = st["kind"], st["case"], st["out"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    if own:
        lib, t, q = st["lib"], st["t"], st["q"]
        rows = (st["cu"].data_ptr(), st["lens"].data_ptr(), len(st["n"]), q.shape[0])
        if kind == "chunk":
            lib.g4_attn_chunk_paged(q.data_ptr(), q.shape[1], t[case["q"]], *_own_pool(st), *rows, case["window"], heads, 1.0,
                                    st["part"].data_ptr(), out.data_ptr(), out.shape[1])
            return out
        k, v, tab = st["k"], st["v"], st["tab"]
        turn = (tab.data_ptr(), tab.shape[0], case["rot"])
        q_in = (q.data_ptr(), q.shape[1], st["qw"].data_ptr(), heads)
        if kind == "post":
            with_kv = case["kv_rows"]
            kv_in = (k.data_ptr(), v.data_ptr(), k.shape[1], st["kw"].data_ptr(), kv) if with_kv else (None, None, 0, None, 0)
            kv_out = (out["k"].data_ptr(), out["v"].data_ptr(), k.shape[1]) if with_kv else (None, None, 0)
            lib.g4_qkv_post_seqs(*q_in, *kv_in, hd, out["q"].data_ptr(), q.shape[1], *kv_out, t[case["q"]], *turn, EPS, *rows)
        else:
            lib.g4_kv_page_append(*_own_pool(st), k.data_ptr(), v.data_ptr(), k.shape[1], st["kw"].data_ptr(), *q_in,
                                  out["q"].data_ptr(), q.shape[1], t[case["q"]], *turn, EPS, *rows)
        return out
    if kind == "chunk":
        page, w = case["page"], case["window"]
        at = 0
        for s, (t, end) in enumerate(zip(st["n"], [a + b for a, b in zip(*_lengths(case))])):
            first = max(0, end - t + 1 - w) if w else 0
            p = torch.arange(first, end, device="cuda")
            pages, slots = st["table"][s][p // page].long(), p % page
            k, v = ((pool[pages, slots].float() if d is None else pool[pages, slots].float() * d[pages, slots])
                    for pool, d in st["pools"])
            last = torch.arange(end - t, end, device="cuda") - first
            seen = (last + 1 - w).clamp(min=0) if w else torch.zeros_like(last)
            out[at:at + t] = _plain_attention(st["q"][at:at + t].reshape(t, heads, hd), k, v, seen, last).reshape(t, -1).to(out.dtype)
            at += t
        return out
    rows = sum(st["n"])
    pages, slots, p = _plain_places(st.get("table"), case.get("page"), st["cu"], st["lens"], rows)
    cs = st["tab"][p]
    for a, h, weight in (("q", heads, st["qw"]), ("k", kv, st["kw"]), ("v", kv, None)):
        if kind == "post" and a not in out:
            continue
        x = _plain_post(st[a][:rows], h, hd, weight, cs)
        if a in out:
            out[a][:rows] = x.reshape(rows, -1).to(out[a].dtype)
        else:
            _put(out[a + "p"], x, pages, slots, a == "v")
    return out


def work(case):
    kind = case["kind"]
    n, had = _lengths(case)
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    rows, q = sum(n), SIZES[case["q"]]
    if kind != "chunk":
        # rows and their (cos, sin) pairs read, results written
        with_kv = kind == "append" or case["kv_rows"]
        kv_size = SIZES[case["type"]] if kind == "append" else q
        once = heads * hd * (4 + q) + (2 * kv * hd * (4 + kv_size) if with_kv else 0) + case["rot"] * 4
        return {"bytes": rows * once, "flops": rows * hd * (10 * heads + (14 * kv if with_kv else 0))}
    row = 2 * kv * (hd * SIZES[case["type"]] + (4 if case["type"] == "Q8" else 0))     # a token's K and V in the cache
    w = case["window"]
    keys = pairs = 0
    for t, h in zip(n, had):
        keys += min(h + t, t - 1 + w) if w else h + t
        whole = max(0, min(t, w - h)) if w else t           # rows that see all before them
        pairs += whole * h + whole * (whole + 1) // 2 + (t - whole) * w
    return {"bytes": keys * row + 2 * q * rows * heads * hd, "flops": 4 * pairs * heads * hd}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the rows themselves
# ---------------------------------------------------------------------------
def _held(x, case):
    """what the cache holds of rows x, in float64"""
    t = case["type"]
    if t != "Q8":
        return x.to(TORCH[t]).double()
    r = x.double().reshape(-1, case["kv"], case["hd"])
    d = (r.abs().max(-1, keepdim=True).values / 127).float().double()
    codes = torch.round((r / d).float().double()).nan_to_num(0.0)
    # a code times its scale is a value of 32 bits
    return (codes * d).float().double().reshape(x.shape)


def _normed(x, heads, hd, weight, pos, tab):
    """heads of rows x in float64: divided by their root mean square, times the weight, each pair a complex number that
    its position's unit turns"""
    x = x.double().view(-1, heads, hd)
    x = x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / hd + EPS) ** 0.5
    if weight is None:
        return x
    x = x * weight.double()
    pairs = torch.complex(x[..., :hd // 2], x[..., hd // 2:])
    unit = torch.ones((len(pos), 1, hd // 2), dtype=torch.complex128, device=x.device)
    unit[:, 0, :tab.shape[1]] = torch.view_as_complex(tab.double().contiguous())[pos]
    pairs = pairs * unit
    return torch.cat([pairs.real, pairs.imag], -1)


def _softmax_rows(q, k, v, first, last):
    """one head in float64: q [rows, hd] over keys first[i]..last[i], in pieces of rows"""
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    kt, v = k.T.contiguous(), v.contiguous()
    at = torch.arange(k.shape[0], device=q.device)
    step = max(1, (1 << 27) // k.shape[0])
    for r in range(0, q.shape[0], step):
        s = q[r:r + step].double() @ kt
        s = s.masked_fill((at < first[r:r + step, None]) | (at > last[r:r + step, None]), -math.inf)
        out[r:r + step] = torch.softmax(s, -1) @ v
    return out


def exact(case, seed):
    kind, hd, heads, kv = case["kind"], case["hd"], case["heads"], case["kv"]
    if kind == "chunk":
        n, had, q, k, v = _chunk_inputs(case, seed)
        k, v = _held(k, case), _held(v, case)
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        w, group, at, key = case["window"], heads // kv, 0, 0
        for t, h in zip(n, had):
            last = h + torch.arange(t, device="cuda")
            first = (last + 1 - w).clamp(min=0) if w else torch.zeros_like(last)
            for i in range(heads):
                c, d = slice(i // group * hd, (i // group + 1) * hd), slice(i * hd, (i + 1) * hd)
                out[at:at + t, d] = _softmax_rows(q[at:at + t, d], k[key:key + h + t, c], v[key:key + h + t, c], first, last)
            at, key = at + t, key + h + t
        return out
    n, had, q, k, v, qw, kw, tab = _post_inputs(case, seed)
    rows = sum(n)
    pos = torch.cat([h + torch.arange(t) for t, h in zip(n, had)]).cuda()
    done = {a: _normed(x[:rows], c, hd, weight, pos, tab)
            for a, x, c, weight in (("q", q, heads, qw), ("k", k, kv, kw), ("v", v, kv, None))}
    out = {}
    for a, x in (("q", q),) + ((("k", k), ("v", v)) if kind == "post" and case["kv_rows"] else ()):
        out[a] = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        out[a][:rows] = done[a].reshape(rows, -1)
    if kind == "append":
        table, pages = _table(case, [a + b for a, b in zip(n, had)], seed)
        seq = torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n)).cuda()
        held = table[seq, pos // case["page"]].long()
        for a, pool in zip("kv", _pools(case, pages)):
            out[a + "p"] = torch.zeros(pool.shape, dtype=torch.float64, device="cuda")
            at = _place(pos % case["page"], hd, pool.element_size(), a == "v")
            block = pos % case["page"] // 16
            for h in range(kv):
                out[a + "p"][held[:, None], h, block[:, None], at] = done[a][:, h]
    return out
