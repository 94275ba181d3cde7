"""Kernels launched while the kernel before them still runs (launch_pdl) wait
for it on every path.  A grid in which no thread waits may end before the one
it depends on, and what follows on the stream is then ordered behind the short
one alone, while the other still uses the workspace."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocketkv-cpp_b200", "csrc")


def _sources():
    out = {}
    for f in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(f) as fh:
            out[os.path.basename(f)] = re.sub(r"//[^\n]*", "", fh.read())
    return out


def _dependents():
    return [(f, k) for f, s in _sources().items() for k in sorted(set(re.findall(r"launch_pdl\(\s*(\w+)", s)))]


def _body(source, kernel):
    at = re.search(r"__global__[^;{]*?\b%s\(" % kernel, source)
    assert at, kernel
    depth, start = 0, source.index("{", at.end())
    for i in range(start, len(source)):
        depth += {"{": 1, "}": -1}.get(source[i], 0)
        if depth == 0:
            return source[start: i]
    raise AssertionError(kernel)


@pytest.mark.parametrize("file,kernel", _dependents(), ids=lambda x: x)
def test_dependent_kernels_wait_before_they_leave(file, kernel):
    body = _body(_sources()[file], kernel)
    wait, leave = body.find("griddepcontrol.wait"), re.search(r"\breturn\b", body)
    assert wait >= 0, "never waits"
    assert leave is None or wait < leave.start(), "a path leaves before the wait"


def test_there_are_such_kernels():
    assert ("sink_attn.cu", "sink_join_kernel") in _dependents() and len(_dependents()) >= 6
