"""The grid of a rotation for every length that is accepted: the header that
the launch uses, compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_grid_covers_the_longest_rows(tmp_path):
    exe = str(tmp_path / "rotary_grid_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-ftrapv", "-x", "c++", os.path.join(ROOT, "tests", "rotary_grid_check.cpp"),
                    "-I" + os.path.join(ROOT, "rocketkv-cpp_b200", "csrc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-3000:]
