"""Argument checks of the 4-bit paged KV cache's entry points, and its plain statement, without a GPU."""
import numpy as np
import pytest

import cactus_b200 as cb
from tests import kv4_util as U

A = 1 << 20  # an aligned address that no refused call touches
GEOM = dict(page=64, hkv=8, d=128, g=32)


def _geom(**kw):
    g = dict(GEOM, **kw)
    return g["page"], g["hkv"], g["d"], g["g"]


def _append(**kw):
    a = dict(k=A, v=A, rs=1024, off=A, lens=A, table=A, ts=4, pool=A, np=10, ps=81920, b=2, t=3)
    a.update({k: v for k, v in kw.items() if k in a})
    return cb.lib().cactus_cuda_kv4_append(a["k"], a["v"], a["rs"], a["off"], a["lens"], a["table"], a["ts"], a["pool"],
                                           a["np"], a["ps"], a["b"], a["t"],
                                           *_geom(**{k: v for k, v in kw.items() if k in GEOM}), None)


def _read(**kw):
    a = dict(pool=A, np=10, ps=81920, table=A, ts=4, off=A, k=A, v=A, b=2, t=3)
    a.update({k: v for k, v in kw.items() if k in a})
    return cb.lib().cactus_cuda_kv4_read(a["pool"], a["np"], a["ps"], a["table"], a["ts"], a["off"], None, a["k"], a["v"],
                                         a["b"], a["t"], *_geom(**{k: v for k, v in kw.items() if k in GEOM}), None)


def _attention(**kw):
    a = dict(q=A, qs=2048, off=A, lens=A, table=A, ts=4, pool=A, np=10, ps=81920, out=A, lse=A, b=2, t=3, mq=2, hq=16,
             scale=0.1, window=0, ws=A, wsb=1 << 40)
    a.update({k: v for k, v in kw.items() if k in a})
    return cb.lib().cactus_cuda_kv4_attention(a["q"], a["qs"], a["off"], a["lens"], a["table"], a["ts"], a["pool"],
                                              a["np"], a["ps"], a["out"], a["lse"], a["b"], a["t"], a["mq"], a["hq"],
                                              *_geom(**{k: v for k, v in kw.items() if k in GEOM}), a["scale"],
                                              a["window"], 1, a["ws"], a["wsb"], None)


def _copy(**kw):
    a = dict(pool=A, np=10, pb=1024, ps=1024, planes=2, pls=10240, src=A, dst=A, n=3)
    a.update(kw)
    return cb.lib().cactus_cuda_kv_copy_pages(a["pool"], a["np"], a["pb"], a["ps"], a["planes"], a["pls"], a["src"],
                                              a["dst"], a["n"], None)


def _compact(**kw):
    a = dict(pool=A, np=10, ps=81920, planes=2, pls=819200, src=A, dst=A, ts=4, kept=A, off=A, b=2, n=3)
    a.update({k: v for k, v in kw.items() if k in a})
    return cb.lib().cactus_cuda_kv4_compact(a["pool"], a["np"], a["ps"], a["planes"], a["pls"], a["src"], a["dst"],
                                            a["ts"], a["kept"], a["off"], a["b"], a["n"],
                                            *_geom(**{k: v for k, v in kw.items() if k in GEOM}), None)


BAD_GEOM = [dict(page=8), dict(page=48), dict(page=512), dict(page=0), dict(hkv=0), dict(hkv=5000), dict(d=96), dict(d=0),
            dict(d=512), dict(g=16), dict(g=0), dict(d=64, g=128)]
BAD_PAGES = [dict(pool=None), dict(pool=A + 8), dict(np=0), dict(np=1 << 32), dict(ps=81904), dict(ps=81928), dict(ts=0),
             dict(ts=1 << 33)]
REFUSED = (
    [(f, k) for f in (_append, _read, _attention, _compact) for k in BAD_GEOM + BAD_PAGES]
    + [(_append, k) for k in (dict(k=None), dict(v=None), dict(off=None), dict(lens=None), dict(table=None),
                              dict(rs=1020), dict(rs=1016), dict(k=A + 2), dict(v=A + 8), dict(t=1 << 31),
                              dict(b=1 << 31))]
    + [(_read, k) for k in (dict(k=None, v=None), dict(off=None), dict(table=None), dict(k=A + 4), dict(v=A + 8),
                            dict(t=1 << 31))]
    + [(_attention, k) for k in (dict(q=None), dict(out=None), dict(ws=None), dict(off=None), dict(lens=None),
                                 dict(table=None), dict(hq=0), dict(hq=12), dict(qs=2040), dict(qs=2052), dict(q=A + 8),
                                 dict(out=A + 8), dict(lse=A + 2), dict(ws=A + 4), dict(wsb=0), dict(scale=0.0),
                                 dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(t=1 << 31),
                                 dict(t=1 << 30, mq=1 << 30, hq=64, qs=8192))]
    + [(_copy, k) for k in (dict(pool=None), dict(src=None), dict(dst=None), dict(np=0), dict(pool=A + 4), dict(pb=1000),
                            dict(ps=1016), dict(pb=2048), dict(pls=100), dict(planes=1 << 17), dict(n=1 << 32))]
    + [(_compact, k) for k in (dict(src=None), dict(dst=None), dict(kept=None), dict(off=None), dict(pls=8),
                               dict(planes=1 << 16), dict(n=1 << 31))]
)


@pytest.mark.parametrize("call,change", REFUSED)
def test_refusals(call, change):
    assert call(**change) == -1
    assert b":" in cb.lib().cactus_cuda_last_error()


def test_empty_calls_do_nothing():
    assert _append(t=0, k=None) == 0 and _append(b=0) == 0
    assert _read(t=0) == 0 and _read(b=0) == 0
    assert _attention(t=0) == 0 and _attention(b=0) == 0 and _attention(mq=0) == 0
    assert _copy(n=0) == 0 and _copy(planes=0) == 0 and _copy(pb=0) == 0
    assert _compact(n=0) == 0 and _compact(planes=0) == 0


def test_page_bytes():
    f = cb.lib().cactus_cuda_kv4_page_bytes
    assert f(64, 8, 128, 32) == 8 * 64 * 2 * (64 + 16) == U.Geom(64, 8, 128, 32).block * 8
    assert f(16, 1, 64, 64) == 16 * 2 * (32 + 4)
    assert f(256, 3, 256, 128) == 3 * 256 * 2 * (128 + 8)
    for bad in BAD_GEOM:
        assert f(*_geom(**bad)) == 0


def test_workspace_is_bounded():
    f = cb.lib().cactus_cuda_kv4_attention_workspace
    assert f(1, 1, 16, 8, 128) >= 16
    assert f(1, 1 << 31, 16, 8, 128) == 0


def test_plain_quantisation_error_is_half_a_step():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)).astype(np.float16)
    q, step, low = U.quantise(x, 32)
    v = U.values(q, step, low, 32).astype(np.float64)
    # half a step, what the step's rounding leaves at the top (15 steps of 2^-10), and fp16's rounding
    bound = np.repeat(step.astype(np.float64), 32, axis=-1) * (0.5 + 15 * 2.0 ** -10) + 2.0 ** -11 * np.abs(v)
    assert np.all(np.abs(v - x.astype(np.float64)) <= bound)


def test_page_map(tmp_path):
    """The handle's bookkeeping (csrc/kv4/page_map.h) against a plain model, with random programs."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "page_map_test")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined",
                    "-I", os.path.join(root, "cactus_b200", "csrc"),
                    os.path.join(root, "tests", "native", "kv4_page_map_test.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


@pytest.mark.parametrize("change", [dict(layers=0), dict(hq=6), dict(hq=0), dict(d=96), dict(page=24), dict(pages=0),
                                    dict(seqs=0), dict(context=0), dict(tokens=0)])
def test_cache_refuses_what_it_cannot_hold(change):
    a = dict(layers=2, hq=8, hkv=4, d=64, g=32, page=16, pages=10, seqs=2, context=100, tokens=8)
    a.update(change)
    L = cb.lib()
    assert not L.cactus_kv4_create(a["layers"], a["hq"], a["hkv"], a["d"], a["g"], a["page"], a["pages"], a["seqs"],
                                   a["context"], a["tokens"], 0)
    assert b"kv4_create" in L.cactus_cuda_last_error()


def test_calls_on_no_cache_are_refused():
    L = cb.lib()
    assert L.cactus_kv4_length(None, 0) == -1 and L.cactus_kv4_truncate(None, 0, 0) == -1
    assert L.cactus_kv4_fork(None, None, None, 0) == -1 and b"null cache" in L.cactus_cuda_last_error()
    L.cactus_kv4_destroy(None)
