"""The steps around the paged cache as the integration notes give them: RoPE
tables filled row by row, norms and rotation over the packed rows, cache and
attention (main.c:1886-1950 of the reference for one sequence), captured; and a
later turn's rows over history read back from the cache."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import paged_np as pn
import test_gpu_paged as base
from test_gpu_paged import Cache, Stream, dbuf, filled, rows, same_bits, within

pytestmark = pytest.mark.gpu

F = C.c_float


@pytest.fixture(scope="module")
def lib():
    from g4 import Lib
    L = Lib.get()
    L.init(0)
    L.L.g4_set_stream(None)
    return L


@pytest.mark.parametrize("hd,n_rot", [(256, 256), (512, 512)])
def test_step_captured(lib, hd, n_rot):
    """One token of every sequence: a g4_rope_table a sequence, at its own device position, then the rows forms, all in
    one graph that is replayed while positions grow; bit for bit the eager calls with tables from host positions, and
    the cache holds the rows that the norms left."""
    rng = np.random.default_rng(700)
    n_heads, n_kv, page, steps = 8, 2, 16, 4
    n = [0, 33, 700, 14]
    s_all, half = len(n), n_rot // 2
    total = [t + steps for t in n]
    table, pages = pn.page_table(rng, total, page)
    hist = rows(rng, sum(n), n_kv, hd)
    raw = [[rows(rng, s_all, h, hd) for h in (n_heads, n_kv, n_kv)] for _ in range(steps)]
    q_norm, k_norm = (dbuf(lib, rng.uniform(0.5, 1.5, hd).astype(np.float32)) for _ in range(2))
    results = []
    for captured in (False, True):
        with Stream(lib):
            c = Cache(lib, rng, pn.F32, hd, n_kv, page, None, table=table, pages=pages)
            c.store(hist, hist, n, n)
            dq, dk, dv = (filled(lib, a.nbytes) for a in raw[0])
            ko, vo, tab = filled(lib, raw[0][1].nbytes), filled(lib, raw[0][1].nbytes), filled(lib, s_all * half * 8)
            out = filled(lib, raw[0][0].nbytes)
            lens, pos, cu = filled(lib, 4 * s_all), filled(lib, 4 * s_all), dbuf(lib, pn.starts([1] * s_all))
            part = filled(lib, lib.L.g4_attn_decode_paged_part_bytes(n_heads, n_kv, hd))

            def run(at=None):
                for s in range(s_all):
                    if at is None:
                        lib.g4_rope_table(tab.ptr + s * half * 8, pos.ptr + 4 * s, 0, n_rot, F(1e4), F(1.0), None)
                    else:
                        lib.g4_rope_table_rows(tab.ptr + s * half * 8, int(at[s]), 1, n_rot, F(1e4), F(1.0), None)
                lib.g4_qkv_post_rows(dq.ptr, q_norm.ptr, dk.ptr, dv.ptr, k_norm.ptr, ko.ptr, vo.ptr, n_kv * hd, tab.ptr, s_all,
                                     n_heads, n_kv, hd, n_rot, F(1e-6))
                lib.g4_kv_page_store(*c.args(), ko.ptr, vo.ptr, n_kv * hd, cu.ptr, lens.ptr, s_all, s_all)
                lib.g4_attn_decode_paged(dq.ptr, n_heads * hd, *c.args(), lens.ptr, s_all, 512, n_heads, F(1.0), part.ptr,
                                         out.ptr, n_heads * hd)

            graph = None
            if captured:
                lib.g4_graph_begin()
                run()
                g = C.c_void_p()
                lib.g4_graph_end(C.byref(g))
                graph = g.value
            got = []
            for i, r in enumerate(raw):
                for d, a in zip((dq, dk, dv), r):
                    d.write(a)
                at = np.array(n, np.int32) + i
                pos.write(at)
                lens.write(at + 1)
                if graph:
                    lib.g4_graph_launch(graph)
                else:
                    run(at)
                lib.g4_sync()
                gk, gv = c.load([1] * s_all, list(at + 1))
                assert same_bits(gk, ko.to_array(np.float32).reshape(gk.shape))
                assert same_bits(gv, vo.to_array(np.float32).reshape(gv.shape))
                got.append(np.concatenate([out.to_array(np.float32), gk.ravel()]))
            results.append(np.stack(got))
            if graph:
                lib.g4_graph_destroy(graph)
    assert np.isfinite(results[0]).all() and same_bits(*results)


@pytest.mark.parametrize("kind,hd", [(pn.BF16, 256), (pn.Q8, 512)])
def test_later_turn(lib, kind, hd):
    """a later turn of one sequence: its history out of the cache into flat rows, its own rows over both, its rows into
    the cache; the next token then sees all of it"""
    rng = np.random.default_rng(710)
    n_heads, n_kv, page, had, new = 8, 2, 16, 100, 37
    c = Cache(lib, rng, kind, hd, n_kv, page, [had + new])
    k, v = rows(rng, had + new, n_kv, hd), rows(rng, had + new, n_kv, hd)
    q = rows(rng, new + 1, n_heads, hd)
    c.store(k[:had], v[:had], [had], [had])
    kc, vc = c.load([had], [had])
    dq, dkc, dvc, dk, dv = (dbuf(lib, x) for x in (q[:new], kc, vc, k[had:], v[had:]))
    out = filled(lib, new * n_heads * hd * 4)
    G = 8
    part = filled(lib, new * lib.L.g4_attn_part_bytes(n_heads, hd, G))
    lib.g4_attn_decode_rows(dq.ptr, dkc.ptr, dvc.ptr, dk.ptr, dv.ptr, n_kv * hd, 0, had, new, 0, n_heads, n_kv, hd, F(0.1), G,
                            part.ptr, out.ptr, None)
    got = out.to_array(np.float32).reshape(new, n_heads, hd)
    hk, hv = (np.concatenate([pn.held(x[:had], kind, hd), x[had:]]).reshape(-1, n_kv, hd) for x in (k, v))
    want, _ = pn.attention(q[:new].reshape(new, n_heads, hd), hk, hv, [0] * new, 0.1)
    assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()      # what the rows form's own tests ask of it
    c.store(k[had:], v[had:], [new], [had + new])
    o = base.run_decode(lib, c, q[new:], [had + new], n_heads, 0, 0.1).reshape(n_heads, hd)
    hk, hv = (pn.held(x, kind, hd).reshape(-1, n_kv, hd) for x in (k, v))
    want, bound = pn.attention(q[new:].reshape(1, n_heads, hd), hk, hv, [0], 0.1)
    within(np.abs(o - want[0]), bound[0], kind)


FIRST = """
import ctypes as C, sys
import numpy as np
sys.path[:0] = {paths!r}
import g4, paged_np as pn, test_gpu_paged as base
lib = g4.Lib.get()
lib.init(0)
with base.Stream(lib):
    rng = np.random.default_rng(720)
    kind, hd, m, n_heads, n_kv = {kind}, {hd}, 300, 8, 2
    q, k, v = (base.cast(base.rows(rng, m, h, hd), kind)[0] for h in (n_heads, n_kv, n_kv))
    dq, dk, dv, cu = (base.dbuf(lib, x) for x in (q, k, v, pn.starts([200, 100])))
    out = base.filled(lib, q.nbytes)
    work = base.filled(lib, lib.L.g4_attn_prompt_packed_work_bytes(kind, 2, m, n_kv, hd))
    call = lambda: lib.g4_attn_prompt_packed(dq.ptr, n_heads * hd, dk.ptr, dv.ptr, n_kv * hd, out.ptr, n_heads * hd, kind,
                                             cu.ptr, 2, m, 0, n_heads, n_kv, hd, C.c_float(0.1), work.ptr)
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
    assert (got[0].reshape(m, -1) != 0x3F).any(1).all()
print("FIRST OK")
"""


@pytest.mark.parametrize("kind,hd", [(pn.F32, 512), (pn.BF16, 256)])
def test_first_call_captured(kind, hd):
    """a process whose first call of the operator is a captured one (kernels with more than 64 KB of LDS)"""
    here = os.path.dirname(os.path.abspath(__file__))
    paths = [here, os.path.join(os.path.dirname(here), "gemma4.c_amd")]
    r = subprocess.run([sys.executable, "-c", FIRST.format(paths=paths, kind=kind, hd=hd)], capture_output=True, text=True,
                       timeout=100)
    assert r.returncode == 0 and "FIRST OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
