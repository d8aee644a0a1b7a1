"""Host side of the 4-bit paged KV cache without a GPU: launch failures, sizes and lists that cannot be."""
import os
import subprocess

import pytest

import cactus_b200 as cb
from cactus_b200 import build

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
