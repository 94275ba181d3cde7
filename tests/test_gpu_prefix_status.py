"""The error word of the shared-prefix decode: what a call recorded stays until
it is looked for, whatever ran behind it, and nothing is found that no call
has recorded."""
import pytest
import torch

import rocketkv_b200 as rkv
from test_gpu_prefix import _query, _setup

pytestmark = pytest.mark.gpu

# (type, D, H, groups, lengths of sequences of no group): every way of a call through the kernels
PLANS = {
    "tensor cores, own tokens joined last": ("bf16", 128, 12, [(256, [260] * 300)], []),
    "tensor cores, three kernels": ("f16", 64, 12, [(1024, [1400] * 20)], []),
    "few rows, one launch": ("bf16", 128, 4, [(1024, [1100] * 3)], []),
    "fp32, many rows": ("f32", 128, 12, [(512, [700] * 20)], []),
    "fp32, own tokens joined last": ("f32", 64, 4, [(128, [130] * 700)], []),
    "no groups": ("bf16", 64, 4, [], [500, 30]),
    "nothing to split": ("bf16", 64, 4, [], [60] * 700),
}


def _call(name, cuda):
    kind, D, H, groups, alone = PLANS[name]
    dt = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[kind]
    cache, starts, shared = _setup(500, 2, D, 16, groups, dt, cuda, alone=alone)
    Q = _query(501, cache.batch, H, D, dt, cuda)
    dec = rkv.PrefixDecoder(H, 2, D, int(cache.lens.max()), cache.batch, dt, cuda, num_groups=len(groups))
    return dec, (Q, cache, starts, shared)


@pytest.mark.parametrize("name", PLANS)
def test_an_error_stays_until_it_is_read(name, cuda):
    dec, args = _call(name, cuda)
    dec(*args)
    assert dec.status() == rkv.RKV_OK
    word = dec.ws[:4].view(torch.int32)
    word.fill_(rkv.RKV_ERR_DEVICE_TIMEOUT)  # as the kernel records it
    for _ in range(3):
        dec(*args)
    assert dec.status() == rkv.RKV_ERR_DEVICE_TIMEOUT
    assert dec.status() == rkv.RKV_OK
    # in a graph, over several replays
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dec(*args)
    word.fill_(rkv.RKV_ERR_DEVICE_TIMEOUT)
    g.replay()
    g.replay()
    assert dec.status() == rkv.RKV_ERR_DEVICE_TIMEOUT
    g.replay()
    assert dec.status() == rkv.RKV_OK
    # a workspace in memory that held anything: not an error
    word.fill_(12345)
    dec(*args)
    assert dec.status() == rkv.RKV_OK


def test_status_of_an_object_whose_only_call_was_captured(cuda):
    """A captured call has not run: its workspace holds what the memory held."""
    warm, args = _call("few rows, one launch", cuda)
    warm(*args)  # loads what a capture must not
    size = warm.ws.numel()
    for fill in (rkv.RKV_ERR_DEVICE_TIMEOUT, 12345):
        junk = [torch.full((size // 4,), fill, dtype=torch.int32, device=cuda) for _ in range(16)]
        del junk  # the new objects' workspaces are likely to lie there
        decs = [rkv.PrefixDecoder(4, 2, 128, warm.max_len, warm.batch, torch.bfloat16, cuda) for _ in range(8)]
        graphs = []
        for dec in decs:
            assert dec.status() == rkv.RKV_OK
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                dec(*args)
        assert [dec.status() for dec in decs] == [rkv.RKV_OK] * len(decs)
        for g in graphs:
            g.replay()
        assert [dec.status() for dec in decs] == [rkv.RKV_OK] * len(decs)
