"""The listing rule of the weight selection on the CPU: the header that the
kernel uses, compiled for the host and walked over whole slices.  A token
listed by two warps would be counted and written twice, behind the end of its
row of kept tokens."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_token_is_listed_once_and_by_its_own_warp(tmp_path):
    exe = str(tmp_path / "weight_list_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-x", "c++", os.path.join(ROOT, "tests", "weight_list_check.cpp"),
                    "-I" + os.path.join(ROOT, "rocketkv-cpp_b200", "csrc"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-3000:]
