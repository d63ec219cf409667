"""Refusals of the operators that branch and trim the cache (no GPU needed), and
the references the GPU tests rely on, against differences and brute force."""

from __future__ import annotations

import itertools

import pytest
import torch

import branch_ref as br


def _rows(b=1, h=2, s=8, d=64, group=32, dtype=torch.bfloat16):
    return br.random_rows(b, h, s, d, group, dtype, 0)


def _tree(**kw):
    from kernels.llama3.tree_attention_quant import tree_attention_quant_gqa
    a = dict(q=torch.zeros(1, 4, 3, 64, dtype=torch.bfloat16), cache=_rows(), draft=_rows(s=3),
             mask=torch.ones(3, 3, dtype=torch.bool), n_q_heads=4, n_kv_heads=2, group_size=32)
    a.update(kw)
    q, cache, draft, mask = a.pop("q"), a.pop("cache"), a.pop("draft"), a.pop("mask")
    return tree_attention_quant_gqa(q, *cache, *draft, mask, **a)


@pytest.mark.parametrize("kw,match", [
    (dict(group_size=0), "group_size"),
    (dict(n_q_heads=0), "must be > 0"),
    (dict(n_q_heads=3), "divisible"),
    (dict(n_q_heads=8), "q head dim"),
    (dict(q=torch.zeros(1, 4, 64, dtype=torch.bfloat16)), "4D"),
    (dict(q=torch.zeros(1, 4, 3, 64, dtype=torch.int32)), "bf16/fp16/fp32"),
    (dict(q=torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16)), "leading dims"),
    (dict(q=torch.zeros(1, 4, 3, 128, dtype=torch.bfloat16)), "too small"),
    (dict(draft=_rows(s=4)), "draft rows"),
    (dict(draft=_rows(s=3, dtype=torch.float32)), "draft scales"),
    (dict(mask=torch.ones(3, 4, dtype=torch.bool)), "tree_mask"),
    (dict(mask=torch.ones(3, 3)), "tree_mask"),
    (dict(), "CUDA"),
])
def test_tree_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        _tree(**kw)


def test_row_refusals():
    from kernels.llama3._checks import check_rows
    k, ks, v, vs = _rows()
    for bad in ((k.float(), ks, v, vs), (k, ks.int(), v, vs), (k, ks, v[:, :, :7], vs),
                (k, ks[:, :, :7], v, vs[:, :, :7]), (k, ks, v, vs.float()), (k[0], ks[0], v[0], vs[0])):
        with pytest.raises(ValueError):
            check_rows("cache", *bad)


def test_commit_refusals():
    from kernels.llama3.tree_attention_quant import commit_draft_rows
    path, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        commit_draft_rows(*_rows(), *_rows(s=3), path, n, context_lens=n)
    with pytest.raises(ValueError, match="match the cache"):
        commit_draft_rows(*_rows(), *_rows(s=3, d=32), path, n, context_lens=n)
    with pytest.raises(ValueError, match="unit stride"):
        strided = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in _rows()]
        commit_draft_rows(*strided, *_rows(s=3), path, n, context_lens=n)


def test_scored_refusals():
    from kernels.llama3.evict import attention_forward_quant_gqa_scored as call
    q, mass = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        call(q, *_rows(), mass, n_q_heads=4, n_kv_heads=2)
    with pytest.raises(ValueError, match="divisible"):
        call(q, *_rows(), mass, n_q_heads=3, n_kv_heads=2)
    with pytest.raises(ValueError, match="group_size"):
        call(q, *_rows(), mass, n_q_heads=4, n_kv_heads=2, group_size=-1)


def test_evict_refusals():
    from kernels.llama3.evict import evict_by_mass
    mass = torch.zeros(1, 2, 8)
    for kw in (dict(keep=9), dict(keep=-1), dict(keep=3, recent=2, sinks=2), dict(keep=4, recent=-1),
               dict(keep=4, sinks=-1)):
        with pytest.raises(ValueError):
            evict_by_mass(*_rows(), mass, **kw)
    with pytest.raises(ValueError, match="CUDA"):
        evict_by_mass(*_rows(), mass, keep=4)


def test_c_abi_refuses_without_touching_a_device():
    """Null pointers, wrong types and shapes come back as statuses."""
    import ctypes

    from kvint4 import _lib, ops
    L = _lib.lib()
    q = torch.zeros(1, 4, 3, 64, dtype=torch.bfloat16)
    cache, draft = _rows(), _rows(s=3)
    mask = torch.ones(3, 3, dtype=torch.uint8)

    def d(t):
        return ctypes.byref(ops.desc(t, host_ok=True))

    def tree(q=q, cache=cache, draft=draft, mask=mask, group=32):
        return L.kv4_tree_attention(d(q), *map(d, cache), *map(d, draft), d(mask), None, d(q), None,
                                    group, 0.0, None, 0, None)

    assert tree(group=0) == _lib.KV4_ERR_INVALID
    assert tree(q=q.to(torch.uint8)) == _lib.KV4_ERR_DTYPE
    assert tree(mask=mask.float()) == _lib.KV4_ERR_DTYPE
    assert tree(mask=mask[:2]) == _lib.KV4_ERR_SHAPE
    assert tree(q=q[:, :3]) == _lib.KV4_ERR_INVALID
    assert tree(draft=_rows(s=3, h=1)) == _lib.KV4_ERR_SHAPE
    assert L.kv4_tree_attention(*[None] * 10, None, None, None, 32, 0.0, None, 0, None) == _lib.KV4_ERR_INVALID
    assert L.kv4_tree_workspace(d(q), *map(d, cache), *map(d, draft), 0) == -_lib.KV4_ERR_INVALID
    assert L.kv4_tree_workspace(d(q), *map(d, cache), *map(d, draft), 32) >= 0
    mass = torch.zeros(1, 2, 8)
    out = _rows(s=4)
    idx = torch.zeros(8, dtype=torch.int32)

    def evict(recent=0, sinks=0, mass=mass, out=out):
        return L.kv4_evict(*map(d, cache), d(mass), *map(d, out), d(torch.zeros(1, 2, out[0].shape[2])),
                           idx.data_ptr(), recent, sinks, None)

    assert evict(recent=3, sinks=2) == _lib.KV4_ERR_INVALID
    assert evict(recent=-1) == _lib.KV4_ERR_INVALID
    assert evict(out=_rows(s=9)) == _lib.KV4_ERR_INVALID
    assert evict(mass=mass.to(torch.float16)) == _lib.KV4_ERR_DTYPE
    assert evict(mass=mass[:, :1]) == _lib.KV4_ERR_SHAPE
    assert L.kv4_scored_attention(*[None] * 8, 32, 1, 1.0, 0.0, None, 0, None) == _lib.KV4_ERR_INVALID
    assert L.kv4_commit_rows(*[None] * 8, None, 0, 0, None, None, None, None) == _lib.KV4_ERR_INVALID


def test_reference_weights_are_the_softmax():
    """The references' own check: weights from the definition, one by one."""
    rows = br.random_rows(1, 1, 6, 8, 4, torch.float32, 1)
    k, v = br.values(*rows[:2], 4, 8)[0], br.values(*rows[2:], 4, 8)[0]
    q = torch.randn(2, 3, 8, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    seen = torch.rand(3, 6, generator=torch.Generator().manual_seed(1)) < 0.6
    seen[1] = False
    out, p, _, _ = br.attend(q, k, v, seen)
    for h, i in itertools.product(range(2), range(3)):
        e = [float(torch.exp(q[h, i] @ k[0, t] / 8 ** 0.5)) if seen[i, t] else 0.0 for t in range(6)]
        total = sum(e)
        for t in range(6):
            assert abs(float(p[h, i, t]) - (e[t] / total if total else 0.0)) < 1e-12
        want = sum((e[t] / total) * v[0, t] for t in range(6)) if total else torch.zeros(8).double()
        assert torch.allclose(out[h, i], want, atol=1e-12)


def test_reference_eviction_by_brute_force():
    mass = torch.tensor([[[3.0, 1.0, 3.0, 0.0, 2.0, 9.0]]])
    assert br.evict_index(mass, 3, 1, 1).tolist() == [[[0, 2, 5]]]
    assert br.evict_index(mass, 4, 0, 0).tolist() == [[[0, 2, 4, 5]]]
    nan = float("nan")
    assert br.evict_index(torch.tensor([[[nan, 1.0, nan, 1.0]]]), 3, 0, 0).tolist() == [[[0, 1, 3]]]


def test_tree_helpers():
    from models.llama3.tree_cache import accept_greedy, tree_depth, tree_mask
    parents = torch.tensor([-1, 0, 0, 1, 3, 2, -1])
    m = tree_mask(parents)
    assert [sorted(torch.nonzero(r).flatten().tolist()) for r in m] == [
        [0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [0, 2, 5], [6]]
    assert tree_depth(parents).tolist() == [0, 1, 1, 2, 3, 2, 0]
    assert torch.equal(tree_mask(torch.stack((parents, parents)))[1], m)
    # tokens: node 0 = 9; children 4, 5; grandchild of 5 is 7
    nodes = torch.tensor([[9, 4, 5, 1, 2, 7, 9], [9, 4, 5, 1, 2, 7, 9]])
    logits = torch.zeros(2, 7, 12)
    logits[0, 0, 5] = logits[0, 2, 7] = logits[0, 5, 11] = 1.0  # 0 -> 5 -> 7 -> 11
    logits[1, 0, 3] = 1.0                                       # nothing fits
    path, accepted, token = accept_greedy(nodes, parents, logits)
    assert accepted.tolist() == [3, 1] and token.tolist() == [11, 3]
    assert path[0, :3].tolist() == [0, 2, 5] and path.dtype == torch.int32


def test_tree_cache_refusals():
    from models.llama3.kv_cache import QuantizedKVCache
    from models.llama3.tree_cache import TreeKVCache
    with pytest.raises(ValueError):
        TreeKVCache(0, 1, 1, 64, capacity=8, max_nodes=4)
    with pytest.raises(ValueError, match="empty"):
        TreeKVCache.from_cache(QuantizedKVCache(), extra=4, max_nodes=4)
    c = TreeKVCache(1, 1, 2, 64, capacity=8, max_nodes=4, device="cpu")
    with pytest.raises(ValueError, match="begin"):
        c.attend(0, torch.zeros(1, 4, 2, 64), torch.zeros(1, 2, 2, 64), torch.zeros(1, 2, 2, 64))
    with pytest.raises(ValueError, match="nodes"):
        c.begin(torch.ones(5, 5, dtype=torch.bool))
    with pytest.raises(ValueError, match="bool"):
        c.begin(torch.ones(2, 2))
    assert c.get_mask_sizes(torch.arange(3)) == (3, 0) and len(c) == 1
    with pytest.raises(ValueError):
        QuantizedKVCache(track_mass=True, mass_window=0)
