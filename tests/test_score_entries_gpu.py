"""Caches that score their tokens: which queries score them does not depend on the
entry that brings them."""

from __future__ import annotations

import pytest
import torch

import branch_ref as br

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


def test_tokens_without_scores_are_not_ranked():
    from models.llama3.kv_cache import QuantizedKVCache
    cache = QuantizedKVCache(track_mass=True, mass_window=16)
    q, k, v = _data(200, 1)
    for layer in (0, 1):  # update: what a module that knows nothing of the scores calls
        cache.update(k[:, :, :150], v[:, :, :150], layer)
    cache.score_window(q[:, :, :150], 0)
    before = [t.clone() for layer in (0, 1) for t in cache.get_quantized(layer)]
    with pytest.raises(ValueError, match="layer 1.*150 tokens"):
        cache.evict(60, recent=8)
    for x, y in zip(before, [t for layer in (0, 1) for t in cache.get_quantized(layer)]):
        assert torch.equal(x, y)  # layer 0 neither
    cache.score_window(q[:, :, :150], 1)
    for layer in (0, 1):
        cache.update(k[:, :, 150:], v[:, :, 150:], layer)
    with pytest.raises(ValueError, match="50 tokens"):
        cache.evict(60, recent=49)
    assert cache.evict(200) == {}
    cache.crop(180)
    assert set(cache.evict(60, recent=30)) == {0, 1}  # the tokens without scores are the recent ones
    with pytest.raises(ValueError, match="30 tokens"):
        cache.evict(40, recent=20)                    # and still have none
    cache.append(k[:, :, :100], v[:, :, :100], 0)     # (grows the buffers)
    with pytest.raises(ValueError, match="130 tokens"):
        cache.evict(70, recent=20)
    cache.crop(30)
    assert set(cache.evict(20)) == {0, 1}


def test_scores_kept_by_hand():
    """Rows appended and scored by the user's own calls are ranked by what stands there."""
    from kernels.llama3.evict import attention_forward_quant_gqa_scored
    from models.llama3.kv_cache import QuantizedKVCache
    cache = QuantizedKVCache(track_mass=True)
    q, k, v = _data(150, 1)
    cache.append(k, v, 0)
    attention_forward_quant_gqa_scored(q[:, :, -8:], *cache.get_quantized(0), cache.mass(0), n_q_heads=8,
                                       n_kv_heads=2, is_causal=True)
    mass = cache.mass(0).cpu()
    kept = cache.evict(40, recent=4)[0].cpu().long()
    assert torch.equal(kept, br.evict_index(mass, 40, 4, 0))


def test_a_masked_prompt_is_not_cut_blindly():
    from transformers import LlamaConfig, LlamaForCausalLM

    from models.llama3.kv_cache import QuantizedKVCache
    from models.llama3.llama3_quant import replace_llama_attention_with_quantized
    torch.manual_seed(0)
    with torch.device("cuda"):
        model = LlamaForCausalLM(LlamaConfig(
            vocab_size=97, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, head_dim=64, tie_word_embeddings=False)).to(torch.bfloat16).eval()
    replace_llama_attention_with_quantized(model)
    ids = torch.randint(0, 97, (2, 40), device="cuda")
    keep = torch.ones_like(ids)
    keep[1, :9] = 0  # padding
    with torch.inference_mode():
        cache = QuantizedKVCache(track_mass=True)
        model(input_ids=ids, past_key_values=cache, use_cache=True, attention_mask=keep)
        with pytest.raises(ValueError, match="no scores"):
            cache.evict(20, recent=4)
        cache = QuantizedKVCache(track_mass=True)
        model(input_ids=ids, past_key_values=cache, use_cache=True)
        assert set(cache.evict(20, recent=4)) == {0, 1}
