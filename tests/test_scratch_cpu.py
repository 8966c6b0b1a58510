"""Who may use the device scratch of the general products, and until when, without a GPU: csrc/scratch.h on a stand-in
for the CUDA runtime."""
import os
import subprocess

from conftest import PKG, ROOT


def test_lifetimes(tmp_path):
    program = str(tmp_path / "scratch_lifetimes")
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-fsanitize=address", "-I", os.path.join(PKG, "csrc"), "-I",
                    os.path.join(cuda, "include"), os.path.join(ROOT, "tests", "native", "scratch_lifetimes.cpp"), "-o",
                    program, "-lpthread"], check=True)
    r = subprocess.run([program], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
