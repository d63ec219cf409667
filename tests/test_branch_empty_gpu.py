"""Tree and scored attention without sequences, queries or tokens."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,group", [(torch.bfloat16, 32), (torch.bfloat16, 16), (torch.float16, 32),
                                         (torch.float32, 32)])
@pytest.mark.parametrize("b,n,s", [(0, 3, 50), (2, 0, 50), (0, 0, 0), (2, 3, 0), (2, 0, 0)])
def test_nothing_to_attend(b, n, s, dtype, group):
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    cache = [t.cuda() for t in br.random_rows(b, 2, s, 128, group, dtype, 1)]
    draft = [t.cuda() for t in br.random_rows(b, 2, n, 128, group, dtype, 2)]
    q = torch.randn(b, 8, n, 128, device="cuda").to(dtype)
    heads = dict(n_q_heads=8, n_kv_heads=2, group_size=group)
    got = tree_attention_quant_gqa(q, *cache, *draft, torch.zeros(n, n, dtype=torch.bool, device="cuda"), **heads)
    assert got.shape == q.shape
    if s == 0:
        assert bool((got == 0).all())
    mass = torch.rand(b, 2, s, device="cuda")
    for causal in (False, True):
        to = torch.full_like(mass, float("nan"))
        out, new = attention_forward_quant_gqa_scored(q, *cache, mass, is_causal=causal, decay=0.5, mass_out=to, **heads)
        torch.cuda.synchronize()
        assert out.shape == q.shape and new is to
        if n == 0:  # no query adds anything
            assert torch.equal(to, 0.5 * mass)
        if s == 0:
            assert bool((out == 0).all())
