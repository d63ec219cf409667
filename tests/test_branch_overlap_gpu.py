"""Overlapping outputs are refused by the compiled entry as well; views that share a
buffer without overlapping are not."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu


def test_one_buffer_for_everything():
    """A capacity buffer that holds cache, drafted rows and eviction's output side by side."""
    from kernels.llama3.evict import attention_forward_quant_gqa_scored, evict_by_mass
    from kernels.llama3.tree_attention_quant import commit_draft_rows, tree_attention_quant_gqa
    b, hq, hkv, s, n, d = 2, 8, 2, 200, 6, 128
    plain = br.random_rows(b, hkv, 2 * s + n, d, 32, torch.bfloat16, 1)
    bufs = [t.cuda() for t in plain]
    cache, draft = [t[:, :, :s] for t in bufs], [t[:, :, s:s + n] for t in bufs]
    room = [t[:, :, s + n:s + n + 50] for t in bufs]
    copies = [[t.clone() for t in x] for x in (cache, draft)]
    q = torch.randn(b, hq, n, d, device="cuda").to(torch.bfloat16)
    mask, heads = torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), dict(n_q_heads=hq, n_kv_heads=hkv)
    want = tree_attention_quant_gqa(q, *copies[0], *copies[1], mask, **heads)
    inplace = q.clone()
    assert torch.equal(tree_attention_quant_gqa(q, *cache, *draft, mask, **heads), want)
    assert torch.equal(tree_attention_quant_gqa(inplace, *cache, *draft, mask, out=inplace, **heads), want)
    masses = torch.rand(b, hkv, s, 2, device="cuda")
    to = torch.empty_like(masses[..., 0])
    out, new = attention_forward_quant_gqa_scored(q, *copies[0], masses[..., 0].contiguous(), mass_out=to, **heads)
    got = attention_forward_quant_gqa_scored(q, *cache, masses[..., 0], mass_out=masses[..., 1], **heads)
    assert torch.equal(got[0], out) and torch.equal(masses[..., 1], new)
    *kept, m, idx = evict_by_mass(*copies[0], new, keep=50, recent=5)
    lens = torch.tensor([0, s - 3], dtype=torch.int32, device="cuda")
    *kept2, m2, idx2 = evict_by_mass(*cache, masses[..., 1], keep=50, recent=5, out=(*room, torch.empty_like(m)))
    assert torch.equal(idx, idx2) and torch.equal(m, m2)
    for x, y in zip(kept, kept2):
        assert torch.equal(x, y)
    path = torch.tensor([[1, 3, 5]] * b, dtype=torch.int32, device="cuda")
    accepted = torch.full((b,), 3, dtype=torch.int32, device="cuda")
    commit_draft_rows(*cache, *draft, path, accepted, context_lens=lens)
    commit_draft_rows(*copies[0], *copies[1], path, accepted, context_lens=lens)
    for x, y in zip(cache, copies[0]):
        assert torch.equal(x, y)


def test_refusals():
    from kernels.llama3.evict import attention_forward_quant_gqa_scored, evict_by_mass
    from kernels.llama3.tree_attention_quant import commit_draft_rows, tree_attention_quant_gqa
    b, hkv, s, n = 1, 2, 100, 4
    cache, draft = ([t.cuda() for t in br.random_rows(b, hkv, t, 64, 32, torch.bfloat16, t)] for t in (s, n))
    before = [t.clone() for t in cache]
    mass = torch.rand(b, hkv, s + 1, device="cuda")
    room = torch.randn(b, 4, n + 1, 64, device="cuda").to(torch.bfloat16)
    q, heads = room[:, :, :n], dict(n_q_heads=4, n_kv_heads=2)
    mask = torch.ones(n, n, dtype=torch.bool, device="cuda")
    ones = torch.ones(3, dtype=torch.int32, device="cuda")
    path = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    for call in (
            lambda: evict_by_mass(*cache, mass[..., :s], keep=9, out=tuple(t[:, :, :9] for t in (*cache, mass))),
            lambda: attention_forward_quant_gqa_scored(q, *cache, mass[..., :s], mass_out=mass[..., 1:], **heads),
            lambda: attention_forward_quant_gqa_scored(q, *cache, mass[:, :1, :s].expand(b, hkv, s), **heads),
            lambda: attention_forward_quant_gqa_scored(q, *cache, mass[..., :s], out=q, **heads),
            lambda: tree_attention_quant_gqa(q, *cache, *draft, mask, out=room[:, :, 1:], **heads),
            lambda: commit_draft_rows(*cache, *[t[:, :, 90:] for t in cache], path, ones[:1], context_lens=ones[1:2]),
            lambda: commit_draft_rows(*cache, *draft, path, ones[:1], context_lens=ones[1:2], lens_out=ones[:1])):
        with pytest.raises(ValueError, match="overlap|expanded"):
            call()
    for x, y in zip(cache, before):
        assert torch.equal(x, y)
