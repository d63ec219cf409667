"""A query that is no number: its rows' outputs and the scores of every token that
it sees are no numbers either, whichever kernel takes the call; other sequences and
KV heads keep theirs."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# kept scores, scores formed again by warps, on tiles, by the kernel for any shape
@pytest.mark.parametrize("dtype,sq,d,group", [(BF16, 1, 128, 32), (F16, 3, 128, 32), (F32, 2, 64, 32),
                                              (BF16, 12, 128, 32), (F16, 12, 64, 64), (BF16, 12, 128, 16),
                                              (BF16, 70, 64, 16), (F32, 12, 64, 32), (BF16, 12, 96, 32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_scores_of_a_query_that_is_no_number(dtype, sq, d, group, bad):
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    b, hq, hkv, s = 2, 8, 2, 300
    cache = [t.cuda() for t in br.random_rows(b, hkv, s, d, group, dtype, 1)]
    q = torch.randn(b, hq, sq, d, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    mass = torch.rand(b, hkv, s, device="cuda")

    def call(x):
        return attention_forward_quant_gqa_scored(x, *cache, mass, n_q_heads=hq, n_kv_heads=hkv, group_size=group,
                                                  is_causal=True, mass_out=torch.empty_like(mass))

    out, new = call(q)
    broken = q.clone()
    broken[1, 5, sq - 1, 7] = bad  # the last query, which sees every token, of KV head 1
    got, scores = call(broken)
    assert torch.equal(scores[0], new[0]) and torch.equal(scores[1, 0], new[1, 0])
    assert torch.equal(got[0], out[0]) and torch.equal(got[1, :5], out[1, :5])
    assert bool(got[1, 5, sq - 1].isnan().all())
    assert bool(scores[1, 1].isnan().all())
