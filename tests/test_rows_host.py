"""What the row operators decide on the host (csrc/rows/ps_rows.hpp), without a
device: tests/rows_host_check.cpp, built for the host alone."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_host_rules(tmp_path):
    out = str(tmp_path / "rows_host_check")
    csrc = os.path.join(ROOT, "powersparse_amd", "csrc")
    subprocess.run([HIPCC, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-Wall",
                    "-I" + os.path.join(ROOT, "include"), "-I" + csrc,
                    "-I" + os.path.join(csrc, "rows"),
                    os.path.join(HERE, "rows_host_check.cpp"), "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
