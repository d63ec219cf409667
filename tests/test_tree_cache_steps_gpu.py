"""TreeKVCache from step to step: a commit takes rows of its own step's tree only."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(tree, n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, hkv = 2, 2
    k, v = (torch.randn(b, hkv, n, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    tree.begin(torch.ones(n, n, dtype=torch.bool, device="cuda").tril())
    tree.attend(0, torch.randn(b, 4, n, 64, device="cuda", generator=g).to(torch.bfloat16), k, v)


def test_rows_of_an_earlier_tree_are_not_committed():
    from kvint4 import ops
    from models.llama3.tree_cache import TreeKVCache
    tree = TreeKVCache(1, 2, 2, 64, capacity=64, max_nodes=8)
    _step(tree, 8, 1)
    tree.commit(torch.tensor([[0, 1]] * 2, dtype=torch.int32, device="cuda"),
                torch.tensor([2, 1], dtype=torch.int32, device="cuda"))
    ops.device_error()
    _step(tree, 3, 2)
    before = [t.clone() for t in tree._cache[0]]
    # node 5 is of the first tree: skipped and reported
    tree.commit(torch.tensor([[0, 5]] * 2, dtype=torch.int32, device="cuda"),
                torch.full((2,), 2, dtype=torch.int32, device="cuda"))
    assert ops.device_error() == 16
    for old, new, draft in zip(before, tree._cache[0], tree._draft[0]):
        for x, at in ((0, 2), (1, 1)):
            assert torch.equal(new[x, :, at], draft[x, :, 0])
            assert torch.equal(new[x, :, at + 1:], old[x, :, at + 1:])


def test_commit_without_a_step():
    from models.llama3.tree_cache import TreeKVCache
    tree = TreeKVCache(1, 2, 2, 64, capacity=64, max_nodes=8)
    path, one = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="begin"):
        tree.commit(path, one)
    _step(tree, 3, 2)
    tree.commit(path, one)
    with pytest.raises(ValueError, match="begin"):
        tree.commit(path, one)
    assert tree.lens.tolist() == [1, 1]


def test_check_reports_a_path_that_does_not_fit():
    from kvint4 import ops
    from models.llama3.kv_cache import QuantizedKVCache
    from models.llama3.tree_cache import TreeKVCache
    ops.device_error()
    tree = TreeKVCache(1, 2, 2, 64, capacity=64, max_nodes=8)
    tree.lens.fill_(tree.capacity - 1)
    _step(tree, 3, 2)
    tree.check()
    path = torch.tensor([[0, 1]] * 2, dtype=torch.int32, device="cuda")
    tree.commit(path, torch.tensor([2, 1], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="accepted count"):
        tree.check()
    tree.check()
    assert tree.lens.tolist() == [tree.capacity - 1, tree.capacity]
    plain = QuantizedKVCache()
    plain.check()
    x = torch.randn(1, 2, 5, 64, device="cuda").to(torch.bfloat16)
    plain.append(x, x, 0)
    plain.check()
