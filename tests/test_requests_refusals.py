"""What the operators of a step over several requests refuse before a kernel
runs: their host code (requests.cpp) built with a driver whose launches
only count themselves (tests/support/requests_refusals.cpp). Host only."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "charlotte_amd", "csrc")


def test_requests_refusals(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no HIP compiler")
    exe = str(tmp_path / "requests_refusals")
    build = subprocess.run([hipcc, "--offload-host-only", "-std=c++17", "-O1", "-g", "-I", CSRC, "-I", os.path.join(ROOT, "include"), "-x",
                            "hip", os.path.join(ROOT, "tests", "support", "requests_refusals.cpp"),
                            os.path.join(CSRC, "requests.cpp"), "-o", exe], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "refused as they should be" in run.stdout, (run.stdout[-3000:], run.stderr[-3000:])
