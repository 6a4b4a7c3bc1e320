"""Host-only AddressSanitizer / UndefinedBehaviorSanitizer builds of the quantised cache's host code, on the CPU: the C
entries' checks, plans and launch sequences (fa_quant_api.cpp) over recording stubs of the launchers."""
import os
import shutil
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "flash-attention-npu_amd", "csrc")
HOST = os.path.join(REPO, "tests", "host")
FLAGS = ["g++", "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
         "-I", CSRC]

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


def build_and_run(tmp_path, *args):
    exe = tmp_path / "check"
    r = subprocess.run([*FLAGS, *args, "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout + r.stderr)[-4000:]
    assert ", 0 failures" in r.stdout, r.stdout


def test_checks_and_plans(tmp_path):
    build_and_run(tmp_path, "-D__HIP_PLATFORM_AMD__=1", "-I", "/opt/rocm/include", "-I", os.path.join(REPO, "include"),
                  os.path.join(CSRC, "fa_quant_api.cpp"), os.path.join(HOST, "fa_quant_host_harness.cpp"))


def test_split_against_brute_force(tmp_path):
    """The decode list's and the prefill line's split (csrc/fa_quant_split.h, host and device code alike): ranges, owners,
    pieces of items and the counts that the merges go by."""
    build_and_run(tmp_path, os.path.join(HOST, "fa_quant_split_check.cpp"))
