"""What kernels need done once on each device (lasp_b200/csrc/per_device.h), with the header that the launchers use; no launcher
keeps the status of a call to the CUDA runtime in a static variable of its own, where a failure would stay for good."""
import glob
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_failure_is_tried_again_and_a_success_is_kept_for_its_device(tmp_path):
    exe = str(tmp_path / "per_device_sim")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "lasp_b200", "csrc"),
                           os.path.join(ROOT, "tests", "csrc", "per_device_sim.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_no_status_is_kept_in_a_static_variable():
    for path in glob.glob(os.path.join(ROOT, "lasp_b200", "csrc", "*.cu*")):
        with open(path) as f:
            assert not re.search(r"\bstatic\s+(const\s+)?cudaError_t\s+\w+\s*=", f.read()), path
