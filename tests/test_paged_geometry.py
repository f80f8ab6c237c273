"""The paged cache's addressing and attention's cut over CTAs, compiled for the
host from the header that the kernels use (no GPU needed)."""
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_paged_geometry(tmp_path):
    exe = str(tmp_path / "paged_check")
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I",
                    os.path.join(HERE, "..", "xingling-cpp_b200", "csrc"), os.path.join(HERE, "paged_check.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
