"""The kernel that lists and packs the rows of a cross entropy call, on the
CPU: its text compiled for the host, each wave once as far ahead of each other
as barriers allow (tests/loss_rows_host.cpp), so that a word of LDS overwritten before a slower
wave has read it gives a wrong list."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "clang++")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no clang++ (vector extensions) in ROCm's llvm/bin")
    out = str(tmp_path_factory.mktemp("loss_rows") / "loss_rows_host")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "hp_rms_norm_amd", "csrc"),
                    os.path.join(ROOT, "tests", "loss_rows_host.cpp"), "-o", out], check=True)
    return out


# up to 512 rows a workgroup takes one; then 2 and 3
@pytest.mark.parametrize("rows,width,stride", [(1, 5, 5), (2, 64, 64), (70, 65, 67), (257, 8, 8),
                                               (700, 9, 11), (1100, 4, 4)])
@pytest.mark.parametrize("ignored", [0, 40, 100])
def test_list_of_rows(program, rows, width, stride, ignored):
    p = subprocess.run([program, str(rows), str(width), str(stride), str(ignored), str(rows + ignored)],
                       capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout == "ok\n", p.stdout + p.stderr


def test_list_of_rows_in_several_passes(program):
    """More than 256 rows a workgroup: the loop over passes reuses its words."""
    p = subprocess.run([program, str(512 * 256 + 300), "1", "1", "40", "3"], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout == "ok\n", p.stdout + p.stderr
