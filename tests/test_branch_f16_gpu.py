"""Half-precision tree attention against the 64-bit result, without the f16
rounding of V in the bound."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,n", [(12, 12, 17), (8, 2, 2), (2, 2, 5)])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 128)])
def test_values_keep_their_f16_scales(hq, hkv, n, d, group):
    """One visible key per row: its weight is 1 whatever the scores, so the output
    is code times scale, which 14 bits hold, rounded once to f16 (bound: U_OUT and
    fp32's u32 for the division by the sum)."""
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    b = 2
    cache = [t.cuda() for t in br.random_rows(b, hkv, 1, d, group, torch.float16, 1)]
    draft = [t.cuda() for t in br.random_rows(b, hkv, n, d, group, torch.float16, 2)]
    q = torch.randn(b, hq, n, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    got = tree_attention_quant_gqa(q, *cache, *draft, torch.eye(n, dtype=torch.bool, device="cuda"),
                                   n_q_heads=hq, n_kv_heads=hkv, group_size=group, context_lens=lens)
    want = br.values(draft[2], draft[3], group, d).repeat_interleave(hq // hkv, 1)
    bound = (br.U_OUT[torch.float16] + 8 * br.U32) * want.abs() + br.TINY[torch.float16]
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
