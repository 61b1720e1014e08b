"""Host arithmetic of the experts' products: launches against the shares that the kernels accept, rows that are copied
against the room reserved for them (csrc/expert_shares.h)."""

import os
import re
import subprocess

from conftest import ROOT


def run_host_program(name, tmp_path):
    exe = tmp_path / name
    cmd = ["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(ROOT, "fsctep_amd", "csrc"),
           os.path.join(ROOT, "tests", "cpp", name + ".cpp"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-3000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-3000:]
    return run.stdout


def test_weight_gradients_launch_the_shares_that_experts_make(tmp_path):
    out = run_host_program("expert_shares", tmp_path)
    cases, equal = map(int, re.search(r"cases (\d+), slots as many as a share (\d+), wrong 0", out).groups())
    assert cases > 10000 and equal > 100
