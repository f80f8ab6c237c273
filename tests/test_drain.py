"""How the products' warps hand accumulators back, also after a wait ran out: the
kernels' own rule, compiled for the host (no GPU needed)."""
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_drain(tmp_path):
    exe = str(tmp_path / "drain_check")
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I",
                    os.path.join(HERE, "..", "xingling-cpp_b200", "csrc"), os.path.join(HERE, "drain_check.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
