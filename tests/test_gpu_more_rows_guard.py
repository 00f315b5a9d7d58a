"""None of layer norm, the router and AdamW writes outside its outputs and workspace: they run in
a child process on buffers of exactly the sizes asked for, with the device allocation guards on
(PS_DEVICE_GUARD: 4 KiB of a known pattern around every block, checked on the host), through
DeviceArray and numpy alone."""
import os
import subprocess
import sys

import pytest

from gpu_util import say

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def test_no_device_write_leaves_its_buffer():
    env = dict(os.environ, PS_DEVICE_GUARD="4096")
    r = subprocess.run([sys.executable, os.path.join(HERE, "more_rows_guard_child.py")], env=env,
                       capture_output=True, text=True, timeout=600)
    say(r.stdout.strip())
    say(r.stderr.strip()[-4000:])
    assert r.returncode == 0, f"child exited with {r.returncode}"
    assert "guard violations: 0" in r.stdout
    assert "ps guard:" not in r.stderr
