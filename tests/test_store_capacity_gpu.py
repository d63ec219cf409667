"""Room of a store that scores its tokens: after an eviction, and as it is reported."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _store(growth, s, capacity=None):
    from kvint4.cache import Int4KVStore
    store = Int4KVStore(32, track_mass=True, growth=growth, capacity=capacity)
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 4, s, 64, generator=g).to(torch.bfloat16).cuda()
    k, v = (torch.randn(2, 2, s, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    store.append(k, v, 0)
    store.score_window(q, 0)
    return store, q, k, v


@pytest.mark.parametrize("growth", [0.25, 1.0, 1.5])
def test_eviction_has_room_for_what_it_keeps(growth):
    store, q, k, v = _store(growth, 1000)
    want, _, _, _ = _store(2.0, 1000)
    kept = store.evict(700, recent=10)[0]
    assert torch.equal(kept, want.evict(700, recent=10)[0])
    layer = store.layer(0)
    assert layer.capacity >= layer.seq_len == 700
    for x, y in zip(layer.views(), want.layer(0).views()):
        assert torch.equal(x, y)
    out = torch.empty_like(q[:, :, :1])
    store.append_attend(q[:, :, :1], k[:, :, :1], v[:, :, :1], 0, out, n_q_heads=4, n_kv_heads=2)
    assert store.layer(0).seq_len == 701


def test_reserved_bytes_count_the_scores():
    store, *_ = _store(1.5, 300, capacity=1024)
    rows = 2 * 2 * 1024
    assert store.capacity_nbytes() == rows * (2 * (32 + 2 * 2) + 4)
    assert store.nbytes() == 2 * 2 * 300 * 2 * (32 + 2 * 2)  # packed rows and scales held
