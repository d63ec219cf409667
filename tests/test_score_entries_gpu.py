"""Caches that score their tokens: which queries score them does not depend on the
entry that brings them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _data(s, seed):
    g = torch.Generator().manual_seed(seed)
    b, hq, hkv, d = 2, 8, 2, 128
    k, v = (torch.randn(b, hkv, s, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    return torch.randn(b, hq, s, d, generator=g).to(torch.bfloat16).cuda(), k, v


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("chunks", [(100,), (2,), (16,), (17, 5), (40, 1, 1, 30)])
def test_append_attend_scores_by_the_window(chunks, causal):
    from kernels.llama3.attention_quant import attention_forward_quant_gqa
    from models.llama3.kv_cache import QuantizedKVCache
    fused, parts = (QuantizedKVCache(track_mass=True, mass_window=16, mass_decay=0.75) for _ in range(2))
    heads = dict(n_q_heads=8, n_kv_heads=2)
    for i, s in enumerate(chunks):
        q, k, v = _data(s, i)
        got = torch.empty_like(q)
        assert fused.append_attend(q, k, v, 0, got, is_causal=causal, **heads) is got
        parts.append(k, v, 0)
        want = attention_forward_quant_gqa(q, *parts.get_quantized(0), group_size=32, is_causal=causal, **heads)
        parts.score_window(q, 0)
        assert float((got.float() - want.float()).abs().max()) < 2e-2
        assert torch.equal(fused.mass(0), parts.mass(0))
    # R heads by the last 16 queries of each chunk, older weight faded
    total = 0.0
    for s in chunks:
        total = 0.75 * total + 4 * min(s, 16)
    assert bool(((fused.mass(0).sum(-1) - total).abs() < 1e-2).all())
