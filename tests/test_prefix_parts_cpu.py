"""What the joins of the shared-prefix decode read where its tcgen05 kernel gave
up a wait and left a row's number of parts and their place unwritten: nothing
behind the buffers.  The header that the kernels use, compiled for the host."""
import glob
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "rocketkv-cpp_b200", "csrc")


def test_parts_lie_in_their_buffer(tmp_path):
    exe = str(tmp_path / "prefix_parts_check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-x", "c++", os.path.join(ROOT, "tests", "prefix_parts_check.cpp"), "-I" + CSRC,
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-3000:]


def test_every_reader_checks_them():
    """The pairs are read in one place, which checks them."""
    reads = []
    for f in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(f) as fh:
            for line in re.sub(r"//[^\n]*", "", fh.read()).splitlines():
                if re.search(r"first_later\[[^=]*$", line):
                    reads.append((os.path.basename(f), line.strip()))
    assert reads and all("parts_behind" in line or f == "prefix.cuh" for f, line in reads), reads
    with open(os.path.join(CSRC, "prefix.cuh")) as fh:
        s = fh.read()
    body = s[s.index("int2 parts_behind("):]
    assert "parts_in_buffer(" in body[: body.index("\n}")]
