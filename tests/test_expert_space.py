"""Host arithmetic of the experts' products: launches against the shares that the kernels accept, rows that are copied
against the room reserved for them (csrc/expert_shares.h)."""

import ctypes
import os
import re
import subprocess

from conftest import ROOT
from fsctep_amd import _lib
from test_experts_host import Dims


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


def test_copies_of_rows_fit_the_room_reserved_for_them(tmp_path):
    out = run_host_program("expert_room", tmp_path)
    cases, copies = map(int, re.search(r"cases (\d+), copies (\d+), wrong 0", out).groups())
    assert cases > 3000 and copies > 3000


def test_fp32_workspaces_hold_no_copies():
    """The workspaces that the C ABI asks for are those of the arrays between the kernels: none for copies in fp32, so none
    may be made there; in bf16 one for each array of rows."""
    lib = _lib.load()

    def sizes(dtype, rows=300, width=64, hidden=40, experts=4, k=2):
        n = [ctypes.c_int64() for _ in range(4)]
        assert lib.fsc_expert_sizes(ctypes.byref(Dims(rows, width, hidden, experts, k, dtype)), *map(ctypes.byref, n)) == 0
        return n[2].value, n[3].value

    a = lambda b: (b + 63) // 64 * 64
    # fp32: h, o, magnitudes of x, h, and the weights' rows
    assert sizes(0)[0] == a(600 * 40 * 4) + a(600 * 64 * 4) + a((300 + 600 + 4 * (80 + 64)) * 4)
    # bf16: h, o, and a copy of x
    assert sizes(1)[0] == a(600 * 40 * 2) + a(600 * 64 * 4) + a(300 * 64 * 2)
