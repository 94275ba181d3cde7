"""The shared-prefix decode under bounds far above what a call holds: max_len,
which decides into how many parts own tokens are cut, and num_groups, which
decides the kernel of the shared ones."""
import pytest
import torch

import rocketkv_b200 as rkv
from test_gpu_prefix import TYPES, _check, _decoder, _query, _setup

pytestmark = pytest.mark.gpu

# (type, D, H, HK, groups, lengths of sequences of no group)
BATCHES = {
    "many sequences": ("bf16", 128, 6, 2, [(272, [272 + 37 * (i % 9) for i in range(150)])], []),   # own tokens fill the GPU under their own max_len
    "some sequences": ("f16", 128, 12, 2, [(1000, [1000 + 41 * i for i in range(30)])], [70, 0]),
    "several groups": ("bf16", 64, 16, 2, [(130, [130, 400, 131]), (512, [600] * 25), (64, [64] * 9)], []),
    "wide": ("bf16", 256, 12, 2, [(300, [310 + i for i in range(24)])], []),
    "few rows": ("f16", 64, 4, 2, [(500, [700, 501])], [300]),
    "fp32": ("f32", 128, 12, 2, [(400, [401 + 50 * i for i in range(12)])], []),
    "fp32, 64 columns": ("f32", 64, 8, 8, [(200, [200, 230, 444])], [1]),
    "no groups": ("bf16", 128, 12, 2, [], [500, 30, 0, 1200]),
}


@pytest.mark.parametrize("top", [12288, 12289, 40000, 131072, 1 << 20, 1 << 30])
@pytest.mark.parametrize("name", BATCHES)
def test_bounds_far_above_the_longest_sequence(name, top, cuda):
    kind, D, H, HK, groups, alone = BATCHES[name]
    dt = TYPES[kind]
    cache, starts, shared = _setup(600, HK, D, 16, groups, dt, cuda, alone=alone)
    Q = _query(601, cache.batch, H, D, dt, cuda)
    dec = _decoder(Q, cache, shared, top)
    dec(Q, cache, starts, shared)
    _check(dec, Q, cache)


@pytest.mark.parametrize("kind,D,HK", [("bf16", 128, 2), ("f16", 64, 2), ("f32", 64, 2), ("bf16", 256, 1)])
def test_one_sequence_with_far_more_own_tokens(kind, D, HK, cuda):
    """More than a part of them holds at most, under a max_len that is cut."""
    dt, B = TYPES[kind], 40
    cache, starts, shared = _setup(610, HK, D, 16, [(256, [30000] + [260 + i for i in range(B - 1)])], dt, cuda)
    Q = _query(611, B, 4 * HK, D, dt, cuda)
    for top in (30000, 65536):
        dec = _decoder(Q, cache, shared, top)
        dec(Q, cache, starts, shared)
        _check(dec, Q, cache)


@pytest.mark.parametrize("kind,D", [("bf16", 128), ("f16", 64), ("bf16", 256), ("f32", 128)])
@pytest.mark.parametrize("capacity", [1, 3, 12, 48, 100])
def test_more_groups_than_are_used(kind, D, capacity, cuda):
    """The same batch under any capacity for groups, the others empty: at its
    end, before it, and with tokens to share."""
    dt, B = TYPES[kind], 48
    cache, starts, shared = _setup(620, 2, D, 16, [(640, [640 + 3 * i for i in range(B)])], dt, cuda)
    Q = _query(621, B, 12, D, dt, cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    dec = rkv.PrefixDecoder(12, 2, D, 800, B, dt, cuda, num_groups=capacity)
    for before, tokens in ((0, 0), (capacity - 1, 0), (capacity // 2, 640)):
        dec.O.fill_(7.0)
        dec.lse.fill_(7.0)
        dec(Q, cache, i32([0] * (before + 1) + [B] * (capacity - before)), i32([tokens] * before + [640] + [tokens] * (capacity - 1 - before)))
        _check(dec, Q, cache)
