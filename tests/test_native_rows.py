"""Whose rows a call on the 8-bit cache has (modgrad_amd/csrc/kv_device.hpp:
kv_seq), compiled for the host: two sequences never have the same row where the
row starts do not overlap, whatever the others hold."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(not os.path.exists(HIPCC) and shutil.which("hipcc") is None,
                    reason="hipcc not available")
def test_rows_of_a_call(tmp_path):
    exe = tmp_path / "rows_check"
    hipcc = HIPCC if os.path.exists(HIPCC) else shutil.which("hipcc")
    subprocess.run([hipcc, "-O2", "-std=c++17", "-x", "hip", "--offload-arch=gfx950", "-o", str(exe),
                    os.path.join(HERE, "native", "rows_check.cpp")], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120,
                       env=dict(os.environ, HIP_VISIBLE_DEVICES=""))  # no device is needed
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok")
