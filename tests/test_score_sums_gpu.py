"""Scores of tokens that receive little: a query's and a head's weights are summed
before they meet the running score, whose rounding they would otherwise each take
(bounds of branch_ref, as in test_evict_gpu)."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hq,sq,s,d,group", [(64, 2, 1500, 64, 64), (64, 2, 1500, 128, 32), (16, 8, 700, 128, 128),
                                             (8, 12, 1500, 96, 32), (32, 40, 700, 128, 32), (64, 20, 700, 64, 16)])
def test_peaked_attention(dtype, hq, sq, s, d, group):
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    b, hkv = 4, 8
    cache = br.random_rows(b, hkv, s, d, group, dtype, 1)
    g = torch.Generator().manual_seed(2)
    q = (3 * torch.randn(b, hq, sq, d, generator=g)).to(dtype)
    mass = 0.5 + 0.5 * torch.rand(b, hkv, s, generator=g)
    _, new = attention_forward_quant_gqa_scored(
        q.cuda(), *[t.cuda() for t in cache], mass.cuda(), n_q_heads=hq, n_kv_heads=hkv, group_size=group,
        is_causal=True, decay=0.5)
    k, v = br.values(*cache[:2], group, d), br.values(*cache[2:], group, d)
    seen = torch.ones(sq, s, dtype=torch.bool).tril(s - sq)
    for x in range(b):
        _, p, X, _ = br.attend(q[x].double(), k[x], v[x], seen)
        add = p.reshape(hkv, -1, s)
        rel = br.weight_bound(X, d, s).reshape(hkv, -1, 1) + br.U32 * (add.shape[1] + 8)
        want = 0.5 * mass[x].double() + add.sum(1)
        bound = (rel * add).sum(1) + br.U32 * 2 * want.abs() + 1e-30
        err = (new[x].cpu().double() - want).abs()
        assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} times the bound"
