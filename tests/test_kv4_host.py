"""Host side of the 4-bit paged KV cache without a GPU: launch failures, sizes and lists that cannot be."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import cactus_b200 as cb
from cactus_b200 import build, kv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_failed_launch_is_an_error(tmp_path):
    """csrc/kv4/kv4_abi.cu linked to launchers that fail, with and without an error of the CUDA runtime."""
    exe = str(tmp_path / "kv4_abi_launch_test")
    subprocess.run([build.nvcc(), build.ARCH, "-std=c++17", "-rdc=true", "--expt-relaxed-constexpr", "-diag-suppress=177",
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "cactus_b200", "csrc"),
                    os.path.join(ROOT, "cactus_b200", "csrc", "kv4", "kv4_abi.cu"),
                    os.path.join(ROOT, "tests", "native", "kv4_abi_launch_test.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr


@pytest.mark.parametrize("change", [dict(layers=1 << 14, pages=1 << 26), dict(layers=65535, pages=(1 << 30) - 1)])
def test_a_pool_of_more_bytes_than_addresses_is_refused(change):
    """2^14 layers of 2^26 pages of 5 * 2^24 bytes are 2^64 bytes five times: none, where the product wraps."""
    L = cb.lib()
    assert L.cactus_cuda_kv4_page_bytes(256, 1024, 256, 32) == 5 << 24
    assert not L.cactus_kv4_create(change["layers"], 1024, 1024, 256, 32, 256, change["pages"], 1, 256, 1, 0)
    assert b"kv4_create: the pool" in L.cactus_cuda_last_error()


@pytest.mark.parametrize("bad", [[0, 2 ** 32 + 1], [-2 ** 31 - 1], np.array([2 ** 40]), [1.5], np.array([2.0]), [None], ["1"],
                                 [True]])
def test_lists_of_the_python_handle_hold_whole_numbers_of_32_bits(bad):
    """Not the rows, or sequences, that the low bits or the whole parts of something else name."""
    with pytest.raises(cb.CactusError, match="whole numbers"):
        kv4._host(bad)


@pytest.mark.parametrize("good", [[], range(3), [2 ** 31 - 1, -2 ** 31], np.arange(4, dtype=np.uint8), np.arange(0), 5,
                                  np.array([[1, 2], [3, 4]], np.int64)])
def test_lists_of_the_python_handle(good):
    a, p = kv4._host(good)
    assert a.dtype == np.int32 and a.tolist() == np.asarray(good).reshape(-1).tolist() and (p.value == a.ctypes.data or not a.size)


def test_a_sequence_number_is_not_cut_to_32_bits():
    cache = kv4.KVCache4.__new__(kv4.KVCache4)
    cache._L, cache.h = cb.lib(), None  # the library answers "null cache"
    for seq, why in ((2 ** 32, "whole numbers"), (1.0, "whole numbers"), (1, "null cache"), (np.int64(1), "null cache")):
        for call in (lambda: cache.length(seq), lambda: cache.truncate(seq, 0), lambda: cache.read(0, seq, 0, 1, 0, 0)):
            with pytest.raises(cb.CactusError, match=why):
                call()
