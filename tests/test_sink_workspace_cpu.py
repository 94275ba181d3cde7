"""The workspace of SinkAttention over calls of changing sizes: host logic, with
the launch left out."""
import pytest
import torch

import rocketkv_b200 as rkv


@pytest.fixture
def launches(monkeypatch):
    """Arguments of the calls that would have been launched."""
    got = []
    monkeypatch.setattr(rkv, "_launch", lambda device, stream, what, fn, *args, **kw: got.append(args))
    monkeypatch.setattr(rkv, "_current_stream", lambda index: 0)
    return got


def _call(att, Lq, Lk=4096, H=8, HK=1, D=128, B=1, **kw):
    Q = torch.empty((B, H, Lq, D), dtype=torch.bfloat16)
    K = torch.empty((B, HK, 1, D), dtype=torch.bfloat16).expand(B, HK, Lk, D)
    return att(Q, K, K, **kw)


def test_lengths_that_rise_step_by_step_keep_a_bounded_workspace(launches):
    """All that is kept for calls in flight stays below twice the largest."""
    att = rkv.SinkAttention(device="cpu")
    for Lq in range(1, 600):
        _call(att, Lq, Lk=32768)
    kept = [t.numel() for t in att._outgrown]
    assert att.ws.numel() > 10 << 20 and sum(kept) <= att.ws.numel()
    for args in launches:  # each call had the workspace that it was told
        assert args[-1] >= 256 and args[-2] != 0


def test_reserved_sizes_do_not_grow_at_the_call(launches):
    att = rkv.SinkAttention(device="cpu")
    att.reserve(rkv.BF16, 8, 1, 128, 300, 32768)
    ws = att.ws
    _call(att, 300, Lk=32768)
    _call(att, 100, Lk=1000)
    assert att.ws is ws and launches[0][-2:] == (ws.data_ptr(), ws.numel())
