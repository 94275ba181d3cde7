"""Waits of the shared-prefix decode's tcgen05 kernel have a limit, all of them:
after one that gave up, the kernel ends.  A named barrier has none, and warps
that meet at one may not agree on whether the wait before it has given up."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rocketkv-cpp_b200", "csrc")


def _kernel():
    with open(os.path.join(CSRC, "prefix_tc.cu")) as f:
        s = re.sub(r"//[^\n]*", "", f.read())
    at = s.index("prefix_tc_kernel(")
    depth, start = 0, s.index("{", at)
    for i in range(start, len(s)):
        depth += {"{": 1, "}": -1}.get(s[i], 0)
        if depth == 0:
            return s[:start], s[start: i]
    raise AssertionError


def test_no_wait_without_a_limit():
    before, body = _kernel()
    for part in (before, body):
        assert not re.search(r"group_sync|group_all|bar\.(sync|red)|(?<!m)barrier\.|try_wait|test_wait|mbar_wait\(", part)
    # the whole CTA's barriers: one before the roles part, one behind them, which every role reaches
    assert body.count("__syncthreads()") == 2
    roles = body[body.index("__syncthreads()") + 15: body.rindex("__syncthreads()")]
    assert "return" not in roles and "warp_wait(&B.pair" in roles
