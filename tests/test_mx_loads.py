"""The direct loads of the MXFP4 tile kernel, walked on the host with the kernel's own address arithmetic."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_no_direct_load_leaves_its_operand(tmp_path):
    """Every tile shape, share of K, ragged end of rows, columns and K, and alignment of the scales."""
    exe = str(tmp_path / "walk")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "litevllm_amd", "csrc"),
                    os.path.join(ROOT, "tests", "mx_span_walk.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout.split()[0]) > 10 ** 6
