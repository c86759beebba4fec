"""Bounded waits of the paged attention kernels and of the sampler that are made to run out: the checker,
tests/cuda/lost_copy_test.cu, compiles the kernels with copies that can be left out, and is compiled here with nvcc. The
call ends without a fault, rows whose work waited for one are NaN (a sampled row: token -1), the others are as before, and
so is the next call."""
import os
import subprocess

import pytest

from conftest import PKG, ROOT

pytestmark = pytest.mark.gpu


def test_waits_that_give_up(cuda, tmp_path):
    src, exe = os.path.join(ROOT, "tests", "cuda", "lost_copy_test.cu"), str(tmp_path / "lost_copy_test")
    subprocess.run(["nvcc", "-std=c++17", "-O3", "-gencode", "arch=compute_100a,code=sm_100a", "-I" + os.path.join(PKG, "csrc"),
                    "-I" + os.path.join(ROOT, "include"), src, "-o", exe], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("\n0 wrong in all"), r.stdout + r.stderr
