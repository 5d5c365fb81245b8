"""Host walk of the dense linear's operand requests (tests/dense_bounds_check.cpp, the address arithmetic of csrc/mx_gemm_addr.h)."""

import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_request_stays_inside_its_operand(tmp_path):
    exe = str(tmp_path / "walk")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", os.path.join(HERE, "dense_bounds_check.cpp"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True)
    assert res.returncode == 0 and "requests inside their operands" in res.stdout, res.stdout
