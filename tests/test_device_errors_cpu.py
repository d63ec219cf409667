"""What the device error word says reaches the caches' users (a stand-in for the
library's word: no GPU needed)."""

from __future__ import annotations

import pytest


def test_check_raises_what_the_word_says(monkeypatch):
    from kvint4 import ops
    from models.llama3.tree_cache import TreeKVCache
    tree = TreeKVCache(1, 1, 2, 64, capacity=8, max_nodes=4, device="cpu")
    word = [0]
    monkeypatch.setattr(ops, "device_error", lambda dev=None: word.pop())
    tree.check()
    for flag, match in ((1, "wait expired"), (8, "scale out of"), (16, "accepted count"), (17, "expired.*; .*path node"),
                        (64, "device error 64")):
        word.append(flag)
        with pytest.raises(RuntimeError, match=match):
            tree.check()
