"""Tree and scored attention in tensor-memory tiles where a CTA's share of the work
holds several short units: sequences of one or two key tiles among long ones, or
nothing but such, with one and two row tiles per unit.  References and bounds as in
test_tree_gpu and test_evict_gpu; the device error word stays clear."""

from __future__ import annotations

import pytest
import torch

from test_evict_gpu import _scored
from test_tree_gpu import _run

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def no_device_error():
    from kvint4 import ops
    ops.device_error()
    yield
    assert ops.device_error() == 0


# heads and nodes: 160, 256, 300 and 320 rows per KV head
@pytest.mark.parametrize("hq,n", [(32, 40), (32, 64), (32, 75), (64, 40)])
@pytest.mark.parametrize("group", [16, 32])
def test_short_sequences_among_long_ones(hq, n, group):
    s = 4096
    _run(8, hq, 8, n, s, 128, group, BF16, lens=[s, 0, 3000, 100, s - 1, 0, 128, 2049], seed=n, want_lse=True)


@pytest.mark.parametrize("hq,n", [(32, 40), (32, 64), (64, 40), (64, 33)])
@pytest.mark.parametrize("d,group", [(128, 32), (64, 16)])
def test_nothing_but_short_sequences(hq, n, d, group):
    g = torch.Generator().manual_seed(n)
    _run(40, hq, 8, n, 128, d, group, BF16, lens=[100] * 40, seed=n)
    for top in (129, 300):
        lens = torch.randint(0, top, (40,), generator=g).tolist()
        _run(40, hq, 8, n, 300, d, group, BF16, lens=lens, seed=top, want_lse=True)


@pytest.mark.parametrize("hq,n", [(32, 40), (64, 40)])
def test_empty_sequences_and_the_same_bits_every_time(hq, n):
    lens = [0 if i % 3 else 700 * (i % 2) + i for i in range(36)]
    want = _run(36, hq, 8, n, 900, 128, 32, BF16, lens=lens, seed=5)
    for _ in range(4):
        assert torch.equal(_run(36, hq, 8, n, 900, 128, 32, BF16, lens=lens, seed=5), want)


@pytest.mark.parametrize("sq", [64, 128])
@pytest.mark.parametrize("hq,d,group", [(64, 128, 32), (32, 64, 16), (24, 128, 128)])
def test_scored_whole_prompts(sq, hq, d, group):
    """Every query is one of the prompt's: no context rows, one key tile per unit."""
    _scored(40, hq, 8, sq, sq, d, group, BF16, causal=True, decay=0.9, seed=sq)
    _scored(24, hq, 8, sq, sq + 70, d, group, BF16, causal=True, decay=0.9, seed=sq + 1)


def test_bad_lengths_among_many():
    from kvint4 import ops
    lens = [900, 901, -1, 900, 1 << 30, 128, 900, 900]
    _run(8, 32, 8, 64, 900, 128, 32, BF16, lens=lens, seed=6)
    assert ops.device_error() == 16
