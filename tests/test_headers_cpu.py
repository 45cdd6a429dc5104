"""The library's headers stand by themselves: included alone, and twice, and with no names outside namespace stk."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "streamtopk-sae_b200", "csrc")


@pytest.mark.skipif(shutil.which("nvcc") is None, reason="no nvcc")
@pytest.mark.parametrize("header,uses", [
    ("stk_vec.cuh", "__device__ unsigned long long f() { return stk::fma2(stk::pair(1.f, 2.f), 0, 0); }\nint pair, halves, fma2;"),
    ("stk_host.h", "bool f() { return stk::aligned_to(nullptr, 4); }\nint aligned_to;")])
def test_header_alone(tmp_path, header, uses):
    src = tmp_path / "alone.cu"
    src.write_text(f'#include "{header}"\n#include "{header}"\n{uses}\n')
    r = subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-c", str(src),
                        "-o", str(tmp_path / "alone.o")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
