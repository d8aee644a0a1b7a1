"""Host side of the 4-bit paged KV cache without a GPU: launch failures, sizes and lists that cannot be."""
import ctypes as C
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


class _Recorded:
    """Stands for the library: keeps what compact is called with, sequences hold 10 rows."""
    rows = None

    def cactus_kv4_length(self, h, seq):
        return 10

    def cactus_kv4_compact(self, h, seqs, rows, offsets, n, stream):
        off = np.ctypeslib.as_array((C.c_int32 * (n + 1)).from_address(offsets.value)).tolist()
        self.rows = [np.ctypeslib.as_array((C.c_int32 * max(1, off[-1])).from_address(rows.value)).tolist()[a:b]
                     for a, b in zip(off, off[1:])]
        return 0

    def cactus_kv4_destroy(self, h):
        pass


def test_slide_keeps_first_and_last_rows_and_refuses_negative_sizes():
    cache = kv4.KVCache4.__new__(kv4.KVCache4)
    cache._L, cache.h = _Recorded(), 1
    for sink, window, kept in ((2, 5, [0, 1, 7, 8, 9]), (0, 3, [7, 8, 9]), (4, 4, [0, 1, 2, 3]), (6, 4, [0, 1, 2, 3]),
                               (3, 50, list(range(10))), (20, 30, list(range(10))), (0, 0, [])):
        cache.slide([0, 1], sink, window)
        assert cache._L.rows == [kept, kept], (sink, window)
    for sink, window in ((0, -1), (-1, 4), (-2, -3)):
        with pytest.raises(cb.CactusError, match="negative"):
            cache.slide([0], sink, window)
