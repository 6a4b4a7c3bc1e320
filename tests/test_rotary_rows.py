"""Rows that the rotation may turn in place (csrc/fa_rotary_rows.h), and the C entry's refusals of the others, on the CPU."""
import os
import shutil
import subprocess

import pytest

from fa_mi355x import capi

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_against_brute_force(tmp_path):
    exe = str(tmp_path / "check")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-I",
                        os.path.join(REPO, "flash-attention-npu_amd", "csrc"), os.path.join(REPO, "tests", "host", "fa_rotary_rows_check.cpp"),
                        "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and ", 0 failures" in r.stdout, (r.stdout + r.stderr)[-4000:]


def call(q, k, heads, heads_k, q_strides, k_strides):
    """fa_rotary in place on a GPU-less machine: the checks run before anything is launched. Pointers are never read: the
    calls here are all refused."""
    f = dict(dtype=1, table_dtype=2, batch=2, seqlen=4, nheads=heads, nheads_k=heads_k, headdim=64, rotary_dim=32, cos=1 << 30, cos_row_stride=16,
             sin=1 << 31, sin_row_stride=16, seqlen_ro=9)
    for name, at, s in (("q", q, q_strides), ("k", k, k_strides)):
        for n in (name, name + "_out"):
            f.update({n: at, n + "_batch_stride": s[0], n + "_row_stride": s[1], n + "_head_stride": s[2]})
    return capi.rotary(**f)


ROW = 6 * 64  # a projection of 4 heads of q, one of k, one of v


@pytest.mark.parametrize("q,k,heads,heads_k,q_strides,k_strides,says", [
    (1 << 20, (1 << 20) + 3 * 128, 4, 2, (4 * ROW, ROW, 64), (4 * ROW, ROW, 64), "same memory"),    # head 3 is of both
    (1 << 20, (1 << 20) + 16, 4, 1, (4 * ROW, ROW, 64), (4 * ROW, ROW, 64), "same memory"),
    (1 << 20, 1 << 20, 4, 4, (4 * ROW, ROW, 64), (4 * ROW, ROW, 64), "same memory"),
    (1 << 20, (1 << 20) + 2 * 4 * ROW - 128, 4, 1, (4 * ROW, ROW, 64), (4 * 64, 64, 64), "same memory"),  # k begins in q's last row
    ((1 << 20) + 128, 1 << 20, 4, 2, (4 * ROW, ROW, 64), (4 * ROW, ROW, 64), "same memory"),
    (1 << 20, 1 << 25, 4, 2, (0, ROW, 64), (4 * ROW, ROW, 64), "repeat rows"),
    (1 << 20, 1 << 25, 4, 2, (4 * ROW, ROW, 64), (4 * ROW, ROW, 32), "repeat rows"),
])
def test_c_entry_refuses(q, k, heads, heads_k, q_strides, k_strides, says):
    assert call(q, k, heads, heads_k, q_strides, k_strides) == capi.FA_EINVAL and says in capi.last_error(), capi.last_error()
