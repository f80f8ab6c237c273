"""What is asked of a device once and kept is that device's own (the library's
header, compiled for the host; no GPU needed)."""
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_per_device(tmp_path):
    exe = str(tmp_path / "per_device_check")
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I",
                    os.path.join(HERE, "..", "xingling-cpp_b200", "csrc"), os.path.join(HERE, "per_device_check.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
