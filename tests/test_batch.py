"""Refusals, sizes and launch failures of a ragged batch's operators (include/cactus_b200_batch.h, the rotating
append of include/cactus_b200_kv4.h), without a GPU: arguments are checked before any CUDA call."""
import os
import subprocess

import pytest

import cactus_b200 as cb
from cactus_b200 import build

A = 1 << 12  # an address that is aligned and never read
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _norm(**kw):
    a = dict(x=A, xs=128, r=A, rs=128, w=A, s=A, ss=128, q=A, sc=A, n=A, rows=4, dims=128, eps=1e-6)
    a.update(kw)
    return cb.lib().cactus_cuda_add_rms_norm_q8(a["x"], a["xs"], a["r"], a["rs"], a["w"], a["s"], a["ss"], a["q"], a["sc"],
                                                a["n"], a["rows"], a["dims"], a["eps"], None)


def _plan(**kw):
    a = dict(off=A, ids=A, s=3, t=50, ad=4, plan=A, pb=1 << 20)
    a.update(kw)
    return cb.lib().cactus_cuda_lora_plan(a["off"], a["ids"], a["s"], a["t"], a["ad"], a["plan"], a["pb"], None)


def _lora(**kw):
    a = dict(x=A, xs=64, a=A, b=A, ranks=A, scales=A, base=2 * A, bs=96, out=A, os=96, plan=A, pb=1 << 20, s=3, t=50, ad=4,
             r=16, k=64, n=96, ws=A, wsb=1 << 24)
    a.update(kw)
    return cb.lib().cactus_cuda_lora_f16(a["x"], a["xs"], a["a"], a["b"], a["ranks"], a["scales"], a["base"], a["bs"],
                                         a["out"], a["os"], a["plan"], a["pb"], a["s"], a["t"], a["ad"], a["r"], a["k"],
                                         a["n"], a["ws"], a["wsb"], None)


def _logits(**kw):
    a = dict(x=A, xs=1000, out=2 * A, os=1000, rows=3, v=1000, pen=A, h=A, ho=A, pl=A, nh=100, bi=A, bv=A, bo=A, nb=10,
             m=A, ms=32, nm=3, mi=A)
    a.update(kw)
    return cb.lib().cactus_cuda_logits_process_f16(a["x"], a["xs"], a["out"], a["os"], a["rows"], a["v"], a["pen"], a["h"],
                                                   a["ho"], a["pl"], a["nh"], a["bi"], a["bv"], a["bo"], a["nb"], a["m"],
                                                   a["ms"], a["nm"], a["mi"], None)


def _table(**kw):
    a = dict(theta=1e4, r=64, p=100, t=A)
    a.update(kw)
    return cb.lib().cactus_cuda_rope_table(a["theta"], a["r"], a["p"], a["t"], None)


def _rope(**kw):
    a = dict(q=A, qs=512, out=2 * A, os=512, k=A, v=A, rs=256, turns=A, np_=100, rot=64, qw=A, kw=A, eps=1e-6, off=A, lens=A,
             table=A, ts=4, pool=A, pages=8, ps=1 << 16, s=2, t=5, hq=8, page=16, hkv=4, d=64, g=32)
    a.update(kw)
    return cb.lib().cactus_cuda_kv4_rope_append(
        a["q"], a["qs"], a["out"], a["os"], a["k"], a["v"], a["rs"], a["turns"], a["np_"], a["rot"], a["qw"], a["kw"],
        a["eps"], a["off"], a["lens"], a["table"], a["ts"], a["pool"], a["pages"], a["ps"], a["s"], a["t"], a["hq"],
        a["page"], a["hkv"], a["d"], a["g"], None)


NAN, INF = float("nan"), float("inf")
REFUSED = (
    [(_norm, k) for k in (dict(x=None), dict(w=None), dict(q=None, n=None), dict(sc=None), dict(rows=1 << 31),
                          dict(dims=32769, xs=40000, rs=40000, ss=40000), dict(xs=127), dict(rs=127), dict(ss=100),
                          dict(xs=1 << 41), dict(rs=1 << 41), dict(ss=1 << 41), dict(ss=136), dict(s=3 * A, x=3 * A, xs=136),
                          dict(eps=-1e-9), dict(eps=NAN), dict(eps=INF), dict(x=A + 1), dict(r=A + 1), dict(w=A + 1),
                          dict(s=A + 1), dict(n=A + 1), dict(sc=A + 2))]
    + [(_plan, k) for k in (dict(off=None), dict(ids=None), dict(plan=None), dict(off=A + 2), dict(ids=A + 1),
                            dict(plan=A + 8), dict(pb=0), dict(s=1 << 31), dict(t=1 << 31), dict(ad=65537))]
    + [(_lora, k) for k in (dict(x=None), dict(a=None), dict(b=None), dict(out=None), dict(plan=None), dict(ws=None),
                            dict(xs=56), dict(bs=88), dict(os=88), dict(xs=68), dict(bs=100), dict(os=100), dict(r=0),
                            dict(r=12), dict(r=264), dict(k=60), dict(n=100, bs=200, os=200), dict(x=A + 8), dict(a=A + 2),
                            dict(b=A + 4), dict(base=A + 8), dict(out=A + 8), dict(plan=A + 4), dict(ws=A + 8),
                            dict(ranks=A + 2), dict(scales=A + 1), dict(base=A, bs=104), dict(pb=64), dict(wsb=64),
                            dict(s=1 << 31), dict(t=1 << 31), dict(ad=1 << 17), dict(xs=1 << 41), dict(k=1 << 21, xs=1 << 21),
                            dict(n=1 << 21, bs=1 << 21, os=1 << 21))]
    + [(_logits, k) for k in (dict(x=None), dict(out=None), dict(rows=1 << 31), dict(v=(1 << 27) + 1, xs=1 << 28, os=1 << 28),
                              dict(xs=999), dict(os=999), dict(out=A, os=1008), dict(ho=None), dict(bv=None), dict(bo=None),
                              dict(ms=31), dict(mi=None, nm=2), dict(nh=1 << 31), dict(nb=1 << 31), dict(nm=1 << 31),
                              dict(x=A + 1), dict(out=A + 1), dict(pen=A + 2), dict(h=A + 2), dict(ho=A + 1), dict(pl=A + 2),
                              dict(bi=A + 2), dict(bv=A + 1), dict(bo=A + 2), dict(m=A + 2), dict(mi=A + 2),
                              dict(xs=1 << 41), dict(os=1 << 41))]
    + [(_table, k) for k in (dict(r=63), dict(t=None), dict(t=A + 8), dict(theta=0.0), dict(theta=-1.0), dict(theta=NAN),
                             dict(theta=INF), dict(p=1 << 40), dict(r=1 << 20))]
    + [(_rope, k) for k in (dict(k=None), dict(v=None), dict(off=None), dict(lens=None), dict(table=None), dict(pool=None),
                            dict(turns=None), dict(np_=0), dict(out=None), dict(rot=72), dict(rot=8), dict(rot=80), dict(eps=-1.0),
                            dict(eps=NAN), dict(hq=0), dict(hq=40000), dict(page=24), dict(d=96), dict(g=48), dict(hkv=0),
                            dict(rs=248), dict(rs=260), dict(qs=504), dict(qs=516), dict(os=504), dict(os=516), dict(q=A + 8),
                            dict(out=A + 8), dict(k=A + 8), dict(v=A + 2), dict(turns=A + 8), dict(qw=A + 8), dict(kw=A + 8),
                            dict(out=A, os=520), dict(s=1 << 31), dict(t=1 << 31), dict(ps=16), dict(ps=(1 << 16) + 8),
                            dict(pages=0), dict(pages=1 << 31), dict(ts=0), dict(pool=A + 8))]
)


@pytest.mark.parametrize("call,change", REFUSED)
def test_refusals(call, change):
    assert call(**change) == -1
    assert b":" in cb.lib().cactus_cuda_last_error()


def test_empty_calls_do_nothing():
    assert _norm(rows=0, x=None) == 0 and _norm(dims=0, w=None) == 0
    assert _plan(s=0, off=None) == 0 and _plan(t=0) == 0
    assert _lora(s=0, x=None) == 0 and _lora(t=0) == 0 and _lora(n=0, bs=0, os=0) == 0
    assert _logits(rows=0, x=None) == 0 and _logits(v=0, xs=0, os=0) == 0
    assert _table(r=0, t=None) == 0 and _table(p=0) == 0
    assert _rope(s=0, k=None) == 0 and _rope(t=0) == 0


def test_sizes_are_bounded():
    L = cb.lib()
    assert L.cactus_cuda_lora_plan_bytes(1, 1, 1) >= 64
    assert L.cactus_cuda_lora_plan_bytes(1 << 31, 1, 1) == 0 and L.cactus_cuda_lora_plan_bytes(1, 1, 1 << 20) == 0
    assert L.cactus_cuda_lora_plan_bytes(1, 1 << 30, 4) == 0  # tokens are below 2^30
    assert L.cactus_cuda_lora_workspace(1000, 64) >= 1000 * 64 * 4
    assert L.cactus_cuda_lora_workspace(1 << 31, 64) == 0 and L.cactus_cuda_lora_workspace(8, 512) == 0
    assert L.cactus_cuda_lora_plan_bytes(4, (1 << 30) - 1, 4) >= 4 << 30  # counted in more than 32 bits


def test_a_failed_launch_is_an_error(tmp_path):
    """batch_abi.cu and rope_abi.cu linked to launchers that fail, with and without an error of the CUDA runtime."""
    exe, src = str(tmp_path / "batch_abi_launch_test"), os.path.join(ROOT, "cactus_b200", "csrc")
    subprocess.run([build.nvcc(), build.ARCH, "-std=c++17", "-rdc=true", "--expt-relaxed-constexpr", "-diag-suppress=177",
                    "-I", os.path.join(ROOT, "include"), "-I", src, os.path.join(src, "batch", "batch_abi.cu"),
                    os.path.join(src, "kv4", "rope_abi.cu"),
                    os.path.join(ROOT, "tests", "native", "batch_abi_launch_test.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


def test_the_first_product_waits_for_what_was_launched_before(tmp_path):
    """lora.cu and lora_tc.cu over a runtime that records their launches, in a thread with programmatic launches on and off."""
    exe, src = str(tmp_path / "lora_launch_test"), os.path.join(ROOT, "cactus_b200", "csrc")
    calls = ("cudaLaunchKernelExC", "cudaGetDevice", "cudaFuncSetAttribute", "cudaGetSymbolAddress")
    subprocess.run([build.nvcc(), build.ARCH, "-std=c++17", "-rdc=true", "--fmad=false", "--expt-relaxed-constexpr",
                    "-diag-suppress=177", "-I", os.path.join(ROOT, "include"), "-I", src,
                    *(o for call in calls for o in ("-Xlinker", "--wrap=" + call)), os.path.join(src, "batch", "lora.cu"),
                    os.path.join(src, "batch", "lora_tc.cu"), os.path.join(ROOT, "tests", "native", "lora_launch_test.cu"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
