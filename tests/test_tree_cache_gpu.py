"""The caches that use the branch and trim operators, and a model that decodes with them."""

from __future__ import annotations

import os
import sys

import pytest
import torch

import branch_ref as br

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BENCH = os.path.join(ROOT, "kv-cache-triton_b200", "benchmarks")


def _tiny(layers=2):
    from transformers import LlamaConfig
    return LlamaConfig(vocab_size=97, hidden_size=256, intermediate_size=256, num_hidden_layers=layers,
                       num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                       max_position_embeddings=4096, initializer_range=0.2, tie_word_embeddings=False)


def test_store_scores_and_evicts():
    from kvint4.cache import Int4KVStore
    store = Int4KVStore(32, track_mass=True)
    g = torch.Generator().manual_seed(0)
    b, hq, hkv, d, s = 2, 8, 2, 128, 150
    k, v = (torch.randn(b, hkv, s, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(b, hq, s, d, generator=g).to(torch.bfloat16).cuda()
    store.append(k, v, 0)
    store.score_window(q, 0)
    assert bool(((store.mass(0).sum(-1) - 4 * 32).abs() < 1e-2).all())  # R heads x 32 queries
    before = [t.clone() for t in store.layer(0).views()]
    mass = store.mass(0).clone()
    kept = store.evict(60, recent=10, sinks=2)[0].cpu().long()
    assert torch.equal(kept, br.evict_index(mass.cpu(), 60, 10, 2))
    for x, y in zip(before, store.layer(0).views()):
        idx = kept.cuda().unsqueeze(-1).expand(-1, -1, -1, x.shape[-1])
        assert torch.equal(y, x.gather(2, idx))
    assert torch.equal(store.mass(0), mass.gather(2, kept.cuda()))
    # decoding goes on: a new token has no score yet, then every token gets its share
    out = torch.empty(b, hq, 1, d, dtype=torch.bfloat16, device="cuda")
    store.append_attend(q[:, :, :1], k[:, :, :1], v[:, :, :1], 0, out, n_q_heads=hq, n_kv_heads=hkv)
    assert store.mass(0).shape[2] == 61
    assert bool(((store.mass(0).sum(-1) - mass.gather(2, kept.cuda()).sum(-1) - 4).abs() < 1e-2).all())
    for _ in range(80):  # growth keeps the scores
        store.append(k[:, :, :1], v[:, :, :1], 0)
    assert bool((store.mass(0)[:, :, 61:] == 0).all()) and float(store.mass(0)[:, :, :60].sum()) > 0
    store.reorder(torch.tensor([1, 0]))
    assert store.evict(200) == {}
    with pytest.raises(ValueError):
        store.evict(3, recent=4)


def test_store_without_scores_refuses_eviction():
    from kvint4.cache import Int4KVStore
    store = Int4KVStore(32)
    x = torch.randn(1, 2, 5, 64, device="cuda").to(torch.bfloat16)
    store.append(x, x, 0)
    with pytest.raises(ValueError, match="track_mass"):
        store.evict(2)


def test_tree_cache_equals_plain_attention():
    """A chain committed node by node is the cache that appending builds."""
    from kernels.llama3.attention_quant import attention_forward_quant_gqa
    from models.llama3.kv_cache import QuantizedKVCache
    from models.llama3.tree_cache import TreeKVCache
    g = torch.Generator().manual_seed(1)
    b, hq, hkv, d, s, n = 2, 8, 2, 128, 70, 5
    k, v = (torch.randn(b, hkv, s + n, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(b, hq, n, d, generator=g).to(torch.bfloat16).cuda()
    plain = QuantizedKVCache()
    plain.append(k[:, :, :s], v[:, :, :s], 0)
    tree = TreeKVCache.from_cache(plain, extra=n, max_nodes=n)
    plain.append(k[:, :, s:], v[:, :, s:], 0)
    tree.begin(torch.ones(n, n, dtype=torch.bool, device="cuda").tril())
    got = tree.attend(0, q, k[:, :, s:], v[:, :, s:])
    want = attention_forward_quant_gqa(q, *plain.get_quantized(0), n_q_heads=hq, n_kv_heads=hkv,
                                       is_causal=True)
    assert float((got.float() - want.float()).abs().max()) < 2e-2
    path = torch.arange(n, dtype=torch.int32, device="cuda").repeat(b, 1)
    tree.commit(path, torch.tensor([n, 2], dtype=torch.int32, device="cuda"))
    assert tree.lens.tolist() == [s + n, s + 2]
    for x, y in zip(tree._cache[0], plain.get_quantized(0)):
        assert torch.equal(x[0, :, :s + n], y[0]) and torch.equal(x[1, :, :s + 2], y[1, :, :s + 2])


@pytest.mark.parametrize("hit", [0.0, 0.6, 1.0])
def test_tree_decoding_gives_the_plain_tokens(hit):
    """fp32, so that both runs choose the same token everywhere."""
    sys.path.insert(0, BENCH)
    from speculative_evict import run
    r = run(batch=3, prompt_len=90, keep=40, steps=17, branch=3, depth=3, hit=hit, seed=5,
            dtype=torch.float32, config=_tiny())
    assert r["layers_cut"] == 2
    assert r["leading_tokens_alike"] == [18] * 3
    assert r["tree_calls"] <= 18 if hit < 1 else r["tree_calls"] <= 6
