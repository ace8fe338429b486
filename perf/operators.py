"""The measured cases of the operators that serve many sequences at once: a
paged KV cache (written, quantised as it is written, and read back), the
attention of one new token of every sequence over it, and the causal attention
of whole prompts packed one after the other.

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


def listed():
    return [
        # 48 conversations store the token they just computed on a global layer
        {"name": "write_tokens", "kind": "write", "type": "Q8", "hd": 512, "heads": 8, "kv": 2, "page": 64, "seqs": 48,
         "lo": 1, "hi": 1, "had": 9000, "pad": 0, "mix": 1},
        # prompts of twelve conversations on a sliding-window layer, some of them later turns; the batch is padded
        {"name": "write_prompts", "kind": "write", "type": "BF16", "hd": 256, "heads": 8, "kv": 2, "page": 16, "seqs": 12,
         "lo": 5, "hi": 2048, "had": 700, "pad": 13, "mix": 2},
        # one conversation's history taken out of the cache, as rows for a prompt that goes on
        {"name": "read_history", "kind": "read", "type": "Q8", "hd": 512, "heads": 8, "kv": 2, "page": 64, "seqs": 1,
         "lo": 3001, "hi": 3001, "pad": 0, "mix": 3},
        # the histories of twenty conversations, moved elsewhere
        {"name": "read_batch", "kind": "read", "type": "F16", "hd": 256, "heads": 8, "kv": 2, "page": 32, "seqs": 20,
         "lo": 17, "hi": 4000, "pad": 7, "mix": 4},
        # the next token of a single short chat, on a sliding-window layer: latency
        {"name": "decode_chat", "kind": "decode", "type": "BF16", "hd": 256, "heads": 8, "kv": 2, "page": 16, "seqs": 1,
         "lo": 203, "hi": 203, "idle": 0, "window": 512, "mix": 5},
        # 64 conversations on a sliding-window layer whose cache keeps the engine's 32 bits
        {"name": "decode_window", "kind": "decode", "type": "F32", "hd": 256, "heads": 8, "kv": 2, "page": 32, "seqs": 64,
         "lo": 1, "hi": 8192, "idle": 0, "window": 512, "mix": 6},
        # one long document on a global layer
        {"name": "decode_long", "kind": "decode", "type": "F16", "hd": 512, "heads": 8, "kv": 2, "page": 64, "seqs": 1,
         "lo": 32768, "hi": 32768, "idle": 0, "window": 0, "mix": 7},
        # a full server: contexts from short to long on a global layer, three slots of the batch unused
        {"name": "decode_batch", "kind": "decode", "type": "Q8", "hd": 512, "heads": 8, "kv": 2, "page": 64, "seqs": 48,
         "lo": 512, "hi": 32768, "idle": 3, "window": 0, "mix": 8},
        # six short messages on a sliding-window layer
        {"name": "prompt_short", "kind": "prompt", "type": "F32", "hd": 256, "heads": 8, "kv": 2, "seqs": 6, "lo": 3, "hi": 60,
         "window": 512, "pad": 0, "mix": 9},
        # nine prompts of ordinary lengths on a sliding-window layer, the batch padded
        {"name": "prompt_window", "kind": "prompt", "type": "F32", "hd": 256, "heads": 8, "kv": 2, "seqs": 9, "lo": 100,
         "hi": 2048, "window": 512, "pad": 11, "mix": 10},
        # three prompts on a global layer, in the engine's 32 bits
        {"name": "prompt_global", "kind": "prompt", "type": "F32", "hd": 512, "heads": 8, "kv": 2, "seqs": 3, "lo": 700,
         "hi": 4096, "window": 0, "pad": 0, "mix": 11},
        # a long document in 16 bits without a window
        {"name": "prompt_long", "kind": "prompt", "type": "BF16", "hd": 256, "heads": 8, "kv": 2, "seqs": 1, "lo": 8191,
         "hi": 8191, "window": 0, "pad": 0, "mix": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "prompt", "prompt"])
    heads, kv = rng.choice([(8, 2), (8, 2), (4, 4), (8, 1), (16, 4), (24, 8), (10, 2), (12, 1), (20, 1), (3, 3)])
    case = {"kind": kind, "type": rng.choice(["F32", "F16", "BF16"] if kind == "prompt" else ["F32", "F16", "BF16", "Q8"]),
            "hd": rng.choice([64, 128, 256, 256, 512, 512]), "heads": heads, "kv": kv, "seqs": _log(rng, 1, 48),
            "mix": rng.randint(0, 10 ** 6)}
    if kind != "prompt":
        case["page"] = rng.choice([16, 32, 64, 128, 256])
    # the tokens of all sequences together: those of an E4B layer in the listed cases, fewer where heads are more or wider
    most = {"write": 12000, "read": 30000, "decode": 300000, "prompt": 8000}[kind]
    if kind == "prompt":
        most = int(most * min(1.0, math.sqrt(4096.0 / (heads * case["hd"]))))
    else:
        most = int(most * min(1.0, 1024.0 / (kv * case["hd"])))
    hi = max(2, min(most // case["seqs"], 8000 if kind == "prompt" else 32768))
    case["hi"] = hi = _log(rng, max(1, hi // 256), hi)
    case["lo"] = _log(rng, 1, hi) if hi > 1 else 1
    if kind == "decode":
        case["idle"] = rng.choice([0, 0, 1, 5])
    else:
        case["pad"] = rng.choice([0, 0, 1, 37])
    if kind == "write":
        case["had"] = rng.choice([0, 1, _log(rng, 2, 4000)])
    if kind in ("decode", "prompt"):
        case["window"] = rng.choice([0, 0, 512, _log(rng, 1, 2000)])
    return case


# ---------------------------------------------------------------------------
# sizes and inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """tokens of each sequence (decode: 0 in the batch's unused slots, spread over it)"""
    rng = random.Random(case["mix"])
    n = [case["lo"] if case["lo"] == case["hi"] else _log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    for _ in range(case.get("idle", 0)):
        n.insert(rng.randint(0, len(n)), 0)
    return n


def _had(case):
    """tokens each sequence of a write has in the cache already"""
    rng = random.Random(case["mix"] + 1)
    return [rng.randint(0, case["had"]) for _ in range(case["seqs"])]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)


def _heads(g, rows, heads, hd, gain=1.0):
    """heads as their norms leave them, of unit rms, a few dims of every head larger; gain: a factor, or one a head"""
    x = torch.randn((rows, heads, hd), device="cuda", generator=g)
    x *= torch.rand((heads, hd), device="cuda", generator=g) * 1.5 + 0.25
    x = x / x.square().mean(-1, keepdim=True).sqrt()
    return (x * gain).reshape(rows, heads * hd)


def _kv(g, rows, case):
    """K (whose norm's weights carry hd^-1/2: the attention scale is 1) and V rows"""
    hd = case["hd"]
    return _heads(g, rows, case["kv"], hd, hd ** -0.5), _heads(g, rows, case["kv"], hd)


def _q(g, rows, case):
    """q rows, from heads that look at everything to heads that look at a few keys"""
    heads = case["heads"]
    return _heads(g, rows, heads, case["hd"], torch.linspace(0.5, 5.0, heads, device="cuda")[:, None])


def _rows(case, seed):
    """(lengths, k, v) of a write or read case: rows of all sequences one after the other, then the padding's"""
    n = _lengths(case)
    k, v = _kv(_gen(seed), sum(n) + case["pad"], case)
    return n, k, v


def _decode_rows(case, seed):
    n = _lengths(case)
    g = _gen(seed)
    q = _q(g, len(n), case)
    return n, q, _kv(g, sum(n), case)


def _prompt_rows(case, seed):
    n = _lengths(case)
    g = _gen(seed)
    rows, t = sum(n) + case["pad"], TORCH[case["type"]]
    q = _q(g, rows, case).to(t)
    k, v = _kv(g, rows, case)
    return n, q, k.to(t), v.to(t)


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
# the plain forms' cache: [pages, page, kv, hd] values or codes, and a scale for each token and head of codes
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


def _plain_places(st):
    """(page, slot) of the rows of a write or a read: the last n of the total tokens of each sequence, one after the other"""
    page, cu = st["case"]["page"], st["cu"].long()
    rows = sum(st["n"])
    seq = torch.repeat_interleave(torch.arange(len(st["n"]), device="cuda"), cu[1:] - cu[:-1], output_size=rows)
    p = torch.arange(rows, device="cuda") + (st["lens"].long() - cu[1:])[seq]
    return st["table"][seq, p // page].long(), p % page


def _plain_store(st, pool, x):
    pages, slots = _plain_places(st)
    codes, d = _plain_encode(x[:sum(st["n"])], st["case"])
    pool[0][pages, slots] = codes
    if d is not None:
        pool[1][pages, slots] = d


def _plain_load(st, pool, out):
    pages, slots = _plain_places(st)
    x = pool[0][pages, slots].float()
    if pool[1] is not None:
        x = x * pool[1][pages, slots]
    out[:len(x)] = x.reshape(len(x), -1)


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
        st["t"] = {"F32": g4.F32, "F16": g4.F16, "BF16": g4.BF16, "Q8": g4.KV_Q8}[case["type"]]
    if kind == "prompt":
        n, st["q"], st["k"], st["v"] = _prompt_rows(case, seed)
        st["out"] = torch.zeros_like(st["q"])
        if own:
            size = lib.L.g4_attn_prompt_packed_work_bytes(st["t"], len(n), st["q"].shape[0], case["kv"], case["hd"])
            st["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        total = n
    else:
        if kind == "decode":
            n, st["q"], (k, v) = _decode_rows(case, seed)
            total = n
            st["out"] = torch.empty_like(st["q"])
        else:
            n, k, v = _rows(case, seed)
            total = [a + b for a, b in zip(n, _had(case))] if kind == "write" else n
            st["out"] = (torch.zeros_like(k), torch.zeros_like(v))
        st["table"], st["pages"] = _table(case, total, seed)
        if own:
            size = lib.L.g4_kv_pool_bytes(st["t"], st["pages"], case["page"], case["kv"], case["hd"])
            st["pools"] = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
            if kind == "decode":
                size = lib.L.g4_attn_decode_paged_part_bytes(case["heads"], case["kv"], case["hd"])
                st["part"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        else:
            st["pools"] = [_plain_pool(case, st["pages"]) for _ in range(2)]
    st.update(n=n, cu=_ints(_starts(n)), lens=_ints(total))
    if kind == "write":
        st.update(k=k, v=v)
    elif kind != "prompt":
        torch.cuda.synchronize()
        if own:
            _own_store(st, k, v)
            lib.g4_sync()
        else:
            for pool, x in zip(st["pools"], (k, v)):
                _plain_store(st, pool, x)
    torch.cuda.synchronize()
    return st


def _own_pool(st):
    """the arguments that name a pool and the pages of its sequences"""
    c = st["case"]
    return (st["pools"][0].data_ptr(), st["pools"][1].data_ptr(), st["t"], st["pages"], c["page"], c["kv"], c["hd"],
            st["table"].data_ptr(), st["table"].shape[1])


def _own_store(st, k, v):
    st["lib"].g4_kv_page_store(*_own_pool(st), k.data_ptr(), v.data_ptr(), k.shape[1], st["cu"].data_ptr(),
                               st["lens"].data_ptr(), len(st["n"]), k.shape[0])


def _own_load(st, k, v):
    st["lib"].g4_kv_page_load(*_own_pool(st), k.data_ptr(), v.data_ptr(), k.shape[1], st["cu"].data_ptr(),
                              st["lens"].data_ptr(), len(st["n"]), k.shape[0])


def run(st):
    kind, case, out = st["kind"], st["case"], st["out"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    if own:
        if kind == "write":
            _own_store(st, st["k"], st["v"])
        if kind in ("write", "read"):
            _own_load(st, *out)
        elif kind == "decode":
            q = st["q"]
            st["lib"].g4_attn_decode_paged(q.data_ptr(), q.shape[1], *_own_pool(st), st["lens"].data_ptr(), q.shape[0],
                                           case["window"], heads, 1.0, st["part"].data_ptr(), out.data_ptr(), out.shape[1])
        else:
            q, k = st["q"], st["k"]
            st["lib"].g4_attn_prompt_packed(q.data_ptr(), q.shape[1], k.data_ptr(), st["v"].data_ptr(), k.shape[1],
                                            out.data_ptr(), out.shape[1], st["t"], st["cu"].data_ptr(), len(st["n"]),
                                            q.shape[0], case["window"], heads, kv, hd, 1.0, st["work"].data_ptr())
    elif kind in ("write", "read"):
        for i, pool in enumerate(st["pools"]):
            if kind == "write":
                _plain_store(st, pool, st["k" if i == 0 else "v"])
            _plain_load(st, pool, out[i])
    elif kind == "decode":
        page, w = case["page"], case["window"]
        for s, t in enumerate(st["n"]):
            if t == 0:
                out[s] = 0.0
                continue
            first = max(0, t - w) if w else 0
            p = torch.arange(first, t, device="cuda")
            pages, slots = st["table"][s][p // page].long(), p % page
            k, v = ((pool[pages, slots].float() if d is None else pool[pages, slots].float() * d[pages, slots])
                    for pool, d in st["pools"])
            none = torch.zeros(1, device="cuda")
            out[s] = _plain_attention(st["q"][s].reshape(1, heads, hd), k, v, none, none + (t - first - 1)).reshape(-1)
    else:
        at = 0
        for t in st["n"]:
            q, k, v = (st[a][at:at + t].reshape(t, -1, hd) for a in "qkv")
            last = torch.arange(t, device="cuda")
            first = (last + 1 - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(last)
            out[at:at + t] = _plain_attention(q, k, v, first, last).reshape(t, -1).to(out.dtype)
            at += t
    return {"k": out[0], "v": out[1]} if kind in ("write", "read") else out


def work(case):
    kind, n = case["kind"], _lengths(case)
    heads, kv, hd, size = case["heads"], case["kv"], case["hd"], SIZES[case["type"]]
    row = 2 * kv * (hd * size + (4 if case["type"] == "Q8" else 0))     # a token's K and V in the cache
    if kind in ("write", "read"):
        # a write reads the rows and stores them; either gives rows of 32 bits
        once = row + 8 * kv * hd
        t = sum(n)
        return {"bytes": t * once * (2 if kind == "write" else 1), "flops": 4 * t * kv * hd}
    w = case["window"]
    if kind == "decode":
        keys = sum(min(w, t) if w else t for t in n)
        return {"bytes": keys * row + 8 * len(n) * heads * hd, "flops": 4 * keys * heads * hd}
    pairs = 0
    for t in n:
        a = min(w, t) if w else t       # rows that see all before them
        pairs += a * (a + 1) // 2 + (t - a) * (w if w else 0)
    return {"bytes": sum(n) * 2 * size * (heads + kv) * hd, "flops": 4 * pairs * heads * hd}


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


def _softmax_rows(q, k, v, first, last):
    """one head in float64: q [rows, hd] over keys first[i]..last[i], in pieces of rows"""
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    kt, v = k.double().T.contiguous(), v.double()
    at = torch.arange(k.shape[0], device=q.device)
    step = max(1, (1 << 27) // k.shape[0])
    for r in range(0, q.shape[0], step):
        s = q[r:r + step].double() @ kt
        s = s.masked_fill((at < first[r:r + step, None]) | (at > last[r:r + step, None]), -math.inf)
        out[r:r + step] = torch.softmax(s, -1) @ v
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind in ("write", "read"):
        n, k, v = _rows(case, seed)
        out = {}
        for name, x in (("k", k), ("v", v)):
            out[name] = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
            out[name][:sum(n)] = _held(x[:sum(n)], case)
        return out
    hd, w, group = case["hd"], case["window"], case["heads"] // case["kv"]
    if kind == "decode":
        n, q, (k, v) = _decode_rows(case, seed)
        k, v = _held(k, case), _held(v, case)
    else:
        n, q, k, v = _prompt_rows(case, seed)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, t in enumerate(n):
        if t == 0:
            continue
        if kind == "decode":
            rows, last = slice(s, s + 1), torch.full((1,), t - 1, device="cuda")
        else:
            rows, last = slice(at, at + t), torch.arange(t, device="cuda")
        first = (last + 1 - w).clamp(min=0) if w else torch.zeros_like(last)
        for h in range(case["heads"]):
            c = slice(h // group * hd, (h // group + 1) * hd)
            out[rows, h * hd:(h + 1) * hd] = _softmax_rows(q[rows, h * hd:(h + 1) * hd], k[at:at + t, c], v[at:at + t, c],
                                                           first, last)
        at += t
    return out
