"""Workspace queries of the branch and trim operators for calls without work: no
sequence, no query, no token.  In a process of their own: a fault on the host would
end it."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kv-cache-triton_b200")

CODE = """
import ctypes
import torch
from kvint4 import _lib, ops
L, (b, n, s) = _lib.lib(), {sizes}
def refs(*ts):
    return [ctypes.byref(ops.desc(t, host_ok=True)) for t in ts]
for dtype in (torch.bfloat16, torch.float16, torch.float32):
    for d, group in ((128, 32), (64, 16)):
        def rows(t):
            return [torch.zeros(b, 2, t, w, dtype=x) for w, x in ((d // 2, torch.uint8), (d // group, dtype)) * 2]
        q = torch.zeros(b, 8, n, d, dtype=dtype)
        print(L.kv4_tree_workspace(*refs(q, *rows(s), *rows(n)), group))
        for causal in (0, 1):
            print(L.kv4_scored_workspace(*refs(q, *rows(s)), group, causal))
"""


@pytest.mark.parametrize("b,n,s", [(0, 3, 50), (2, 0, 50), (0, 0, 0), (2, 3, 0), (2, 0, 0)])
def test_workspace_of_calls_without_work(b, n, s):
    r = subprocess.run([sys.executable, "-c", CODE.format(sizes=(b, n, s))], capture_output=True, text=True,
                       cwd=PKG, timeout=300)
    assert r.returncode == 0, r.stderr[-400:]
    sizes = [int(x) for x in r.stdout.split()]
    assert len(sizes) == 18 and all(x >= 0 for x in sizes)
    if b * n == 0:
        assert not any(sizes)
