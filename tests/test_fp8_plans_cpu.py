"""Plans of the 8-bit products for devices that are not there."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "venom_b200")


def test_plans_belong_to_their_device(tmp_path):
    from venom_b200 import build
    build.build_lib()
    exe = str(tmp_path / "plans")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", "/usr/local/cuda/include", "-o", exe, os.path.join(ROOT, "tests", "fp8_plans_check.cpp"), "-L" + PKG, "-lvenom_b200",
                           "-L/usr/local/cuda/lib64", "-lcudart", "-pthread", "-Wl,-rpath," + PKG, "-Wl,-rpath,/usr/local/cuda/lib64"])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "plans ok" in r.stdout, (r.returncode, r.stdout, r.stderr)
